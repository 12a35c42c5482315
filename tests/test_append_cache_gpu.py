"""Writing the cache on the GPU: which slots change and to what, which stay, and what is refused or left out."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import Cache, assert_turned, randn, turn

pytestmark = pytest.mark.gpu

FREQ = [1e6 ** (-i / 64) for i in range(64)]
AXIS = [0] * 16 + [1] * 24 + [2] * 24


def snapshot(cache):
    return cache.k.clone(), cache.v.clone()


@pytest.mark.parametrize("page,layout", [(0, "plain"), (0, "heads"), (8, "plain"), (16, "pairs"), (48, "layers"), (64, "heads"), (256, "plain")])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("lens,counts", [([0], [1]), ([5, 0, 63, 64], [1, 1, 1, 1]), ([7, 120, 0], [90, 0, 301]), ([1000] * 2, [700, 333])])
def test_slots(page, layout, turned, lens, counts):
    gen = torch.Generator().manual_seed(sum(lens) + page)
    kvh, qh = 2, 6
    cache = Cache(page, len(lens), max(n + c for n, c in zip(lens, counts)) + 3, kvh, page, layout)
    before = snapshot(cache)
    total = sum(counts)
    uniform = len(set(counts)) == 1
    shape = (len(lens), counts[0]) if uniform else (total,)
    k, v, q = (randn(gen, *shape, h, 128).cuda() for h in (kvh, kvh, qh))
    cu = None if uniform else torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
    more, ref_k = {}, k.cpu().reshape(-1, kvh, 128).double()
    if turned:
        positions = torch.randint(0, 10**6, (3, *shape), generator=gen)
        more = dict(q=q, positions=positions.cuda(), axes=min_fa3_op.RotaryAxes(FREQ, AXIS))
        ref_k = turn(ref_k, positions.reshape(3, -1), FREQ, AXIS, False)
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    q_out = min_fa3_op.append_cache(k, v, cache.k, cache.v, lens_d, block_table=cache.table, cu_seqlens=cu, **more)
    min_fa3_op.check_last_status("append_cache")
    assert lens_d.tolist() == lens
    if turned:
        flat = q.cpu().reshape(-1, qh, 128)
        assert_turned(q_out.reshape(flat.shape), flat, turn(flat, positions.reshape(3, -1), FREQ, AXIS, False), 64)
    else:
        assert q_out is None
    untouched = torch.ones(cache.k.shape[:2], dtype=torch.bool)
    first = 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        pages, rows = cache.index(b, n, n + c)
        untouched[pages, rows] = False
        got_k, got_v = cache.rows("k", b, n + c)[n:], cache.rows("v", b, n + c)[n:]
        assert torch.equal(got_v, v.cpu().reshape(-1, kvh, 128).double()[first:first + c])
        if c:
            assert_turned(got_k, k.cpu().reshape(-1, kvh, 128)[first:first + c], ref_k[first:first + c], 64)
        if not turned:
            assert torch.equal(got_k, ref_k[first:first + c])
        first += c
    for new, old in zip((cache.k, cache.v), before):
        assert torch.equal(new.cpu()[untouched], old.cpu()[untouched]), "slots of others changed"


def test_padding_rows_go_nowhere():
    # A batch padded for a captured graph: rows behind the last sequence are not written and not turned.
    gen = torch.Generator().manual_seed(1)
    cache = Cache(3, 2, 64, 2, 16)
    before = snapshot(cache)
    k, v, q = (randn(gen, 12, h, 128).cuda() for h in (2, 2, 4))
    cu = torch.tensor([0, 3, 5], dtype=torch.int32).cuda()
    lens = torch.tensor([10, 20], dtype=torch.int32).cuda()
    positions = torch.zeros(1, 12, dtype=torch.int32).cuda()
    out = min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, block_table=cache.table, cu_seqlens=cu, q=q,
                                  positions=positions, axes=min_fa3_op.RotaryAxes.from_sections((64,)))
    min_fa3_op.check_last_status("append_cache")
    assert torch.equal(out[:5], q[:5])
    changed = (cache.k != before[0]).any(-1).any(-1)
    assert int(changed.sum()) == 5


def test_more_sequences_than_a_warp():
    gen = torch.Generator().manual_seed(2)
    counts = [i % 3 for i in range(100)]
    cache = Cache(4, 100, 40, 1, 8)
    k, v = randn(gen, sum(counts), 1, 128).cuda(), randn(gen, sum(counts), 1, 128).cuda()
    cu = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
    lens = torch.arange(100, dtype=torch.int32) % 37
    min_fa3_op.append_cache(k, v, cache.k, cache.v, lens.cuda(), block_table=cache.table, cu_seqlens=cu)
    min_fa3_op.check_last_status("append_cache")
    first = 0
    for b, c in enumerate(counts):
        n = int(lens[b])
        assert torch.equal(cache.rows("k", b, n + c)[n:], k[first:first + c].double().cpu())
        first += c


@pytest.mark.parametrize("what", ["beyond the slots", "negative length", "page too high", "negative page"])
def test_what_has_no_place_is_left_out_and_reported(what):
    gen = torch.Generator().manual_seed(5)
    cache = Cache(6, 2, 64, 2, 16)
    before = snapshot(cache)
    lens = [10, 20]
    if what == "beyond the slots":
        lens[1] = 63                                      # tokens 64 and 65 have no slot
    elif what == "negative length":
        lens[1] = -2
    else:
        cache.table[1, 1] = cache.k.size(0) if what == "page too high" else -1
    k, v = randn(gen, 2, 3, 2, 128).cuda(), randn(gen, 2, 3, 2, 128).cuda()
    min_fa3_op.append_cache(k, v, cache.k, cache.v, torch.tensor(lens, dtype=torch.int32).cuda(), block_table=cache.table)
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("append_cache")
    assert torch.equal(cache.rows("k", 0, 13)[10:], k[0].double().cpu())
    changed = (cache.k != before[0]).any(-1).any(-1)
    assert int(changed.sum()) == {"beyond the slots": 4, "negative length": 4}.get(what, 3)
    # The next call's status is its own.
    min_fa3_op.append_cache(k, v, cache.k, cache.v, torch.tensor([0, 0], dtype=torch.int32).cuda(), block_table=cache.table)
    min_fa3_op.check_last_status("append_cache")


def test_graph_with_changing_lengths():
    gen = torch.Generator().manual_seed(7)
    cache = Cache(8, 3, 64, 2, 16)
    k, v = randn(gen, 3, 1, 2, 128).cuda(), randn(gen, 3, 1, 2, 128).cuda()
    lens = torch.tensor([0, 5, 15], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, block_table=cache.table)
        lens.add_(1)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        k.copy_(randn(gen, 3, 1, 2, 128))
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate((0, 5, 15)):
            assert torch.equal(cache.rows("k", b, n + step + 1)[-1:], k[b].double().cpu())
