"""Eviction against a plain statement of its rules: which slots stay, where they go, ties, lengths, layouts, overlaps."""
from __future__ import annotations

import math

import pytest
import torch

import min_fa3_op
from cache_util import Cache

pytestmark = pytest.mark.gpu


def order(weights, n, budget, recent):
    """For one head: the slot that each of the first slots of the result comes from."""
    if n <= budget:
        return list(range(n))
    old = budget - recent
    def rank(j):
        w = weights[j]
        return (0, 0.0, j) if math.isnan(w) else (1, -w, j)
    best = sorted(range(n - recent), key=rank)[:old]
    late = iter(sorted(j for j in best if j >= old))
    stay = {j for j in best if j < old}
    return [j if j in stay else next(late) for j in range(old)] + list(range(n - recent, n))


def check(cache, weights, lens, budget, recent, call_weights=None):
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    before_k, before_v = cache.k.clone().cpu(), cache.v.clone().cpu()
    w = weights.cuda() if call_weights is None else call_weights
    new_lens, new_weights, index = min_fa3_op.evict_cache(cache.k, cache.v, w, lens_d, budget, recent=recent,
                                                          block_table=cache.table)
    min_fa3_op.check_last_status("evict_cache")
    assert lens_d.tolist() == lens and torch.equal(w.cpu().nan_to_num(nan=7.25), weights.nan_to_num(nan=7.25))
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    want_k, want_v = before_k.clone(), before_v.clone()
    for b, n in enumerate(lens):
        m = min(n, budget)
        pages, rows = cache.index(b)
        for h in range(cache.kvh):
            place = order(weights[b, h].tolist(), n, budget, recent)
            assert index[b, h, :m].tolist() == place, (b, h)
            assert (index[b, h, m:] == -1).all() and not new_weights[b, h, m:].any()
            assert torch.equal(new_weights[b, h, :m].cpu().nan_to_num(nan=7.25), weights[b, h][place].nan_to_num(nan=7.25))
            at = torch.tensor(place, dtype=torch.long)
            want_k[pages[:m], rows[:m], h] = before_k[pages[at], rows[at], h]
            want_v[pages[:m], rows[:m], h] = before_v[pages[at], rows[at], h]
    # Behind the new length, the slots keep what they had.
    assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)
    return new_lens, new_weights, index


def draw(seed, *shape):
    gen = torch.Generator().manual_seed(seed)
    w = torch.rand(*shape, generator=gen) ** 4 * 50
    return torch.where(torch.rand(*shape, generator=gen) < 0.1, torch.zeros(()), w)


@pytest.mark.parametrize("page,layout", [(0, "plain"), (0, "heads"), (8, "layers"), (16, "pairs"), (48, "plain"), (128, "heads")])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (60, 0), (60, 7), (60, 60), (300, 100), (511, 300), (512, 64)])
def test_budgets_and_layouts(page, layout, budget, recent):
    lens = [513, 60, 0, 61, 512]
    cache = Cache(budget + page, len(lens), 520, 2, page, layout)
    check(cache, draw(budget, len(lens), 2, cache.slots), lens, budget, recent)


@pytest.mark.parametrize("n,budget,recent", [(4097, 4096, 64), (4097, 4096, 4096), (5000, 3000, 2500), (40000, 9999, 1), (40000, 39990, 333),
                                             (33, 32, 31), (1025, 1024, 0), (100000, 1000, 10)])
def test_long_sequences(n, budget, recent):
    cache = Cache(n, 2, n, 1, 64)
    check(cache, draw(n, 2, 1, cache.slots), [n, max(1, n // 3)], budget, recent)


def test_ties_go_to_the_lower_slot():
    cache = Cache(1, 1, 1000, 4, 16)
    weights = torch.zeros(1, 4, cache.slots)
    weights[0, 1] = 3.5                                     # all equal
    weights[0, 2] = (torch.arange(cache.slots) % 3).float()
    weights[0, 3, ::2] = -0.0                               # as large as 0
    check(cache, weights, [1000], 400, 20)


def test_infinities_nan_negative_and_tiny_weights():
    cache = Cache(2, 1, 300, 2, 16)
    weights = draw(3, 1, 2, cache.slots) - 20
    weights[0, 0, 100:110], weights[0, 0, 200], weights[0, 0, 50:60] = float("nan"), float("inf"), float("-inf")
    weights[0, 1, :290] = torch.arange(290) * 2.0**-149     # below the smallest normal number
    check(cache, weights, [300], 30, 5)


def test_what_lies_behind_a_sequence_does_not_matter():
    cache = Cache(4, 1, 300, 1, 16)
    weights = draw(5, 1, 1, cache.slots)
    weights[..., 250:] = float("nan")
    check(cache, weights, [250], 100, 10)


def test_strided_weights_with_fewer_slots_than_the_cache():
    cache = Cache(6, 2, 600, 2, 16)
    weights = draw(7, 2, 2, 301)
    wide = torch.zeros(2, 3, 2, 400).cuda()
    view = wide[:, 1, :, 50:351]
    view.copy_(weights)
    check(cache, weights, [301, 290], 200, 30, call_weights=view)


def test_again_and_again():
    """Decoding with a budget: the cache grows by some slots and is cut back."""
    cache = Cache(8, 2, 140, 2, 8)
    lens, weights = [100, 37], draw(9, 2, 2, cache.slots)
    for step in range(6):
        lens_d, weights_d, _ = check(cache, weights, lens, 90, 16)
        weights = weights_d.cpu()
        lens = [n + 5 + step for n in lens_d.tolist()]
        for b, n in enumerate(lens):
            weights[b, :, :n] += draw(step + 20, 2, n)


@pytest.mark.parametrize("what", ["too long", "negative length", "page too high", "negative page"])
def test_what_does_not_exist_is_left_out_and_reported(what):
    cache = Cache(10, 2, 64, 1, 16)
    weights = draw(11, 2, 1, cache.slots)
    lens = [40, 60]
    if what == "too long":
        lens[1] = 65
    elif what == "negative length":
        lens[1] = -1
    else:
        cache.table[1, 2] = cache.k.size(0) if what == "page too high" else -3
    before = cache.k.clone()
    out = min_fa3_op.evict_cache(cache.k, cache.v, weights.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 20, recent=4,
                                 block_table=cache.table)
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("evict_cache")
    place = order(weights[0, 0].tolist(), 40, 20, 4)
    assert out[2][0, 0].tolist() == place
    pages, rows = cache.index(0)
    assert torch.equal(cache.k.cpu()[pages[:20], rows[:20]], before.cpu()[pages[torch.tensor(place)], rows[torch.tensor(place)]])


@pytest.mark.parametrize("recent", [0, 4])
@pytest.mark.parametrize("what", ["too long", "negative length", "page too high", "negative page"])
def test_what_does_not_exist_where_many_rows_move(what, recent):
    """As above, with rows moved by launches of their own."""
    cache = Cache(14, 2, 1280, 1, 16)
    weights = draw(15, 2, 1, cache.slots)
    lens = [900, 1200]
    if what == "too long":
        lens[1] = cache.slots + 1
    elif what == "negative length":
        lens[1] = -1
    else:
        cache.table[1, 2] = cache.k.size(0) if what == "page too high" else -3
    before = cache.k.cpu()
    out = min_fa3_op.evict_cache(cache.k, cache.v, weights.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 200, recent=recent,
                                 block_table=cache.table)
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("evict_cache")
    place = torch.tensor(order(weights[0, 0].tolist(), 900, 200, recent))
    assert torch.equal(out[2][0, 0].cpu().long(), place)
    pages, rows = cache.index(0)
    assert torch.equal(cache.k.cpu()[pages[:200], rows[:200]], before[pages[place], rows[place]])


@pytest.mark.parametrize("seqs", [252, 253, 300])
def test_many_sequences(seqs):
    """Up to 252 sequences report in words of their own."""
    cache = Cache(seqs, seqs, 24, 1, 8)
    check(cache, draw(seqs, seqs, 1, cache.slots), [(b * 7) % 25 for b in range(seqs)], 11, 3)


@pytest.mark.parametrize("budget", [48, 49, 1000])
def test_a_budget_that_no_sequence_exceeds(budget):
    cache = Cache(budget, 2, 48, 2, 16)
    check(cache, draw(budget, 2, 2, cache.slots), [48, 0], budget, min(budget, 20))


def test_graph_and_another_stream():
    cache = Cache(12, 2, 200, 2, 16)
    weights, lens = draw(13, 2, 2, cache.slots).cuda(), torch.tensor([200, 150], dtype=torch.int32).cuda()
    start_k, start_v = cache.k.clone(), cache.v.clone()
    want = min_fa3_op.evict_cache(cache.k, cache.v, weights, lens, 100, recent=10, block_table=cache.table)
    want_k = cache.k.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = min_fa3_op.evict_cache(cache.k, cache.v, weights, lens, 100, recent=10, block_table=cache.table)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        cache.k.copy_(start_k)
        cache.v.copy_(start_v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(cache.k, want_k)
