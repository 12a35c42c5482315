"""Writing a cache in 8 bits on the GPU: which slots and scales change and to what, which stay, and what is refused or left out.

Tolerances.  Values that are not turned are divided by powers of two and rounded once: equal bits.  Turned values are off by 2^-20 of
the largest before they are rounded (as in the tests of ``rotary``), which may tip a rounding to either side: they are within half a
step of e4m3 (2^-4 of the value, or half of 2^-9 of the scale) and that of the value in 64 bits, and their scale is the smallest that
holds the block's largest value, give or take as much."""
from __future__ import annotations

import math

import pytest
import torch

import min_fa3_op
from cache8_util import E4M3, E4M3_HALF_STEP, E4M3_SMALLEST, Cache8, scale_for, write
from cache_util import assert_turned, randn, turn

pytestmark = pytest.mark.gpu

FREQ = [1e6 ** (-i / 64) for i in range(64)]
AXIS = [0] * 16 + [1] * 24 + [2] * 24


def held(cache, which, b, n):
    """One sequence's e4m3 values [slots, heads, 128] and scales [blocks, heads], in 64 bits."""
    pages = torch.tensor([p for p, _ in cache.place[b][:n]], dtype=torch.long)
    rows = torch.tensor([r for _, r in cache.place[b][:n]], dtype=torch.long)
    values = getattr(cache, which).view(torch.uint8).cpu()[pages, rows].view(E4M3).double()
    return values, getattr(cache, which + "_scales").cpu().double()[pages, rows // cache.block][::cache.block]


def check(cache, before, which, b, first, new, n):
    """``new`` [tokens, heads, 128] written from slot ``first`` on, values that were not turned."""
    values, scales = held(cache, which, b, n)
    for h in range(cache.kvh):
        want, want_scales = write(before[0][:, h], before[1][:, h], first, new[:, h], cache.block)
        assert torch.equal(scales[:, h], want_scales), f"scales of sequence {b}, head {h}"
        same = (values[:, h] == want) | (values[:, h].isnan() & want.isnan())
        assert same.all(), f"{which} of sequence {b}, head {h}: {int((~same).sum())} values differ"


def call(cache, k, v, lens, **more):
    out = min_fa3_op.append_cache(k, v, cache.k, cache.v, torch.tensor(lens, dtype=torch.int32).cuda(), **cache.more(), **more)
    min_fa3_op.check_last_status("append_cache")
    return out


@pytest.mark.parametrize("page,block,layout", [(0, 16, "plain"), (0, 128, "heads"), (16, 16, "pairs"), (48, 16, "layers"), (64, 32, "heads"),
                                               (64, 64, "plain"), (256, 128, "pairs"), (128, 16, "plain")])
@pytest.mark.parametrize("lens,counts", [([0], [1]), ([5, 0, 63, 64], [1, 1, 1, 1]), ([7, 120, 0], [90, 0, 301]), ([1000] * 2, [700, 333]),
                                         ([17, 130], [3, 3])])
def test_slots_and_scales(page, block, layout, lens, counts):
    gen = torch.Generator().manual_seed(sum(lens) + page)
    cache = Cache8(page, len(lens), max(n + c for n, c in zip(lens, counts)) + 3, 2, page, block, layout)
    uniform, total = len(set(counts)) == 1, sum(counts)
    shape = (len(lens), counts[0]) if uniform else (total,)
    # Tokens of different sizes, so that scales grow in the middle of blocks, and some do not.
    sizes = torch.exp2(torch.randint(-6, 7, (*shape, 2, 1), generator=gen).float()).to(torch.bfloat16)
    k, v = randn(gen, *shape, 2, 128) * sizes, randn(gen, *shape, 2, 128) * sizes.flip(-2)
    before = {(w, b): held(cache, w, b, cache.slots) for w in "kv" for b in range(len(lens))}
    snapshot = cache.snapshot()
    cu = None if uniform else torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
    call(cache, k.cuda(), v.cuda(), lens, cu_seqlens=cu)
    flat = {"k": k.reshape(-1, 2, 128).double(), "v": v.reshape(-1, 2, 128).double()}
    first = 0
    mine = torch.zeros(cache.k.shape[0], dtype=torch.bool)
    for b, (n, c) in enumerate(zip(lens, counts)):
        mine[torch.tensor([p for p, _ in cache.place[b]])] = True
        for which in "kv":
            check(cache, before[which, b], which, b, n, flat[which][first:first + c], cache.slots)
        first += c
    for new, old in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scales, cache.v_scales), snapshot):
        assert torch.equal(new.cpu()[~mine], old.cpu()[~mine]), "pages of nobody changed"


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("pairs", [8, 32, 64])
@pytest.mark.parametrize("block,count", [(16, 1), (16, 40), (64, 30), (128, 300)])
def test_turned(adjacent, pairs, block, count):
    gen = torch.Generator().manual_seed(pairs + count)
    lens, freq, axis = [3, 150], FREQ[:pairs], AXIS[:pairs]
    axis[-1] = 2
    cache = Cache8(pairs, 2, 500, 2, 128, block)
    q, k, v = randn(gen, 2, count, 6, 128), randn(gen, 2, count, 2, 128), randn(gen, 2, count, 2, 128)
    # Blocks that new tokens begin inside of have large scales, which those keep.
    for scales in (cache.k_scales, cache.v_scales):
        scales.fill_(0.25)
    positions = torch.randint(0, 10**6, (3, 2, count), generator=gen)
    axes = min_fa3_op.RotaryAxes(freq, axis, adjacent=adjacent, magnitude=1.25)
    out = call(cache, k.cuda(), v.cuda(), lens, q=q.cuda(), positions=positions.cuda(), axes=axes)
    flat = positions.reshape(3, -1)

    def turned(x):
        ref = turn(x.reshape(-1, x.size(-2), 128), flat, freq, axis, adjacent)
        if adjacent or pairs < 64:
            ref[..., :2 * pairs] *= 1.25
        else:
            ref *= 1.25
        return ref

    assert_turned(out.reshape(-1, 6, 128), q.reshape(-1, 6, 128), turned(q), pairs)
    ref = turned(k).view(2, count, 2, 128)
    for b, n in enumerate(lens):
        got = cache.rows("k", b, n + count)[n:]
        scales = held(cache, "k", b, n + count)[1]
        slack = 2**-20 * 1.25 * k.double().abs().max().item()
        for j in range(n // block, (n + count - 1) // block + 1):
            lo, hi = max(n, j * block), min(n + count, (j + 1) * block)
            for h in range(2):
                here, scale = ref[b, lo - n:hi - n, h], scales[j, h].item()
                most = here.abs().max().item()
                if lo > j * block:
                    assert scale == 0.25
                else:
                    assert scale in (scale_for(most + slack), scale_for(most - slack))
                off = (got[lo - n:hi - n, h] - here).abs()
                assert (off <= here.abs() * E4M3_HALF_STEP + scale * E4M3_SMALLEST / 2 + slack * 1.1).all()


def test_token_by_token_and_at_once():
    """A block filled token by token ends with the scale of its largest token, and values that were rounded at most once more each time
    the scale grew: exact but for those that became the smallest of the format."""
    gen = torch.Generator().manual_seed(3)
    k = randn(gen, 1, 50, 2, 128) * torch.exp2(torch.arange(50) / 5.0).view(1, 50, 1, 1).to(torch.bfloat16)
    v = randn(gen, 1, 50, 2, 128)
    one, all_ = (Cache8(4, 1, 64, 2, 64, 32) for _ in range(2))
    for t in range(50):
        call(one, k[:, t:t + 1].cuda(), v[:, t:t + 1].cuda(), [t])
    call(all_, k.cuda(), v.cuda(), [0])
    assert torch.equal(one.k_scales.cpu()[all_.table.cpu()[0, 0]], all_.k_scales.cpu()[all_.table.cpu()[0, 0]])
    a, b = one.rows("k", 0, 50), all_.rows("k", 0, 50)
    scale = held(all_, "k", 0, 50)[1].repeat_interleave(32, 0)[:50, :, None]
    assert ((a - b).abs() <= scale * E4M3_SMALLEST).all()
    assert torch.equal(one.rows("v", 0, 50).isfinite(), all_.rows("v", 0, 50).isfinite())


@pytest.mark.parametrize("block", [16, 64])
def test_zeros_infinities_nan_and_the_ends_of_the_range(block):
    gen = torch.Generator().manual_seed(5)
    cache = Cache8(6, 1, 64, 1, 64, block)
    k = randn(gen, 1, 48, 1, 128)
    k[0, :16] = 0
    k[0, 16:32, 0, 5] = math.inf
    k[0, 17, 0, 6], k[0, 18, 0, 7] = -math.inf, math.nan
    k[0, 32:] *= torch.exp2(torch.linspace(-126, -60, 16)).view(16, 1, 1).to(torch.bfloat16)
    v = k.flip(1) * 2.0**100
    before = {w: held(cache, w, 0, cache.slots) for w in "kv"}
    call(cache, k.cuda(), v.cuda(), [0])
    for which, new in (("k", k), ("v", v)):
        check(cache, before[which], which, 0, 0, new[0].double(), cache.slots)


def test_largest_values_on_the_border():
    """448 times a power of two fits exactly; the next bf16 does not."""
    cache = Cache8(7, 1, 32, 1, 32, 16)
    k = torch.zeros(1, 32, 1, 128, dtype=torch.bfloat16)
    k[0, 3, 0, 0], k[0, 20, 0, 0] = 448 * 2.0**-5, 450 * 2.0**-5
    call(cache, k.cuda(), k.cuda(), [0])
    page = cache.table.cpu()[0, 0]
    assert cache.k_scales.cpu()[page, :, 0].tolist() == [2.0**-5, 2.0**-4]


def test_scales_of_another_maker_are_kept_while_they_are_enough():
    gen = torch.Generator().manual_seed(8)
    cache = Cache8(9, 1, 64, 2, 64, 64, powers=False)
    cache.k_scales.fill_(0.0123)
    cache.v_scales.fill_(1e-4)
    before = {w: held(cache, w, 0, 64) for w in "kv"}
    k, v = randn(gen, 1, 5, 2, 128), randn(gen, 1, 5, 2, 128)
    call(cache, k.cuda(), v.cuda(), [20])
    page = cache.table.cpu()[0, 0]
    assert (cache.k_scales.cpu()[page] == torch.tensor(0.0123)).all()
    got = cache.rows("k", 0, 25)[20:]
    assert ((got - k[0].double()).abs() <= k[0].double().abs() * E4M3_HALF_STEP * (1 + 2**-20) + 0.0123 * E4M3_SMALLEST / 2 * (1 + 2**-20)).all()
    # V's had to grow: those that were there are divided by a ratio that is no power of two, in 32 bits, and rounded again.
    scale = cache.v_scales.cpu().double()[page][0]
    assert all(math.frexp(s)[0] == 0.5 for s in scale.tolist())
    old, now = before["v"][0][:20] * before["v"][1][0][:, None], cache.rows("v", 0, 20)
    assert ((now - old).abs() <= old.abs() * E4M3_HALF_STEP * (1 + 2**-20) + scale[:, None] * E4M3_SMALLEST / 2 * (1 + 2**-20)).all()


def test_padding_rows_go_nowhere():
    gen = torch.Generator().manual_seed(1)
    cache = Cache8(3, 2, 64, 2, 16)
    snapshot = cache.snapshot()
    k, v, q = (randn(gen, 12, h, 128).cuda() for h in (2, 2, 4))
    k[5:], v[5:] = 1e6, 1e6
    cu = torch.tensor([0, 3, 5], dtype=torch.int32).cuda()
    positions = torch.zeros(1, 12, dtype=torch.int32).cuda()
    out = call(cache, k, v, [10, 20], cu_seqlens=cu, q=q, positions=positions, axes=min_fa3_op.RotaryAxes.from_sections((64,)))
    assert torch.equal(out[:5], q[:5])
    assert cache.k_scales.max().item() <= max(snapshot[2].max().item(), 2.0)


def test_more_sequences_than_a_warp():
    gen = torch.Generator().manual_seed(2)
    counts = [i % 4 for i in range(100)]
    cache = Cache8(4, 100, 48, 1, 16)
    k, v = randn(gen, sum(counts), 1, 128), randn(gen, sum(counts), 1, 128)
    cu = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
    lens = [i % 43 for i in range(100)]
    before = [held(cache, "k", b, cache.slots) for b in range(100)]
    call(cache, k.cuda(), v.cuda(), lens, cu_seqlens=cu)
    first = 0
    for b, c in enumerate(counts):
        check(cache, before[b], "k", b, lens[b], k[first:first + c].double(), cache.slots)
        first += c


@pytest.mark.parametrize("what", ["beyond the slots", "negative length", "page too high", "negative page"])
def test_what_has_no_place_is_left_out_and_reported(what):
    gen = torch.Generator().manual_seed(5)
    cache = Cache8(6, 2, 64, 2, 16)
    before = {b: held(cache, "k", b, 64) for b in range(2)}
    snapshot = cache.snapshot()
    lens = [10, 20]
    if what == "beyond the slots":
        lens[1] = 63                                      # tokens 64 and 65 have no slot
    elif what == "negative length":
        lens[1] = -2
    else:
        cache.table[1, 1] = cache.k.size(0) if what == "page too high" else -1
    k, v = randn(gen, 2, 3, 2, 128), randn(gen, 2, 3, 2, 128)
    k[1, 1:] *= 1000
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    min_fa3_op.append_cache(k.cuda(), v.cuda(), cache.k, cache.v, lens_d, **cache.more())
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("append_cache")
    check(cache, before[0], "k", 0, 10, k[0].double(), 64)
    changed = (cache.k.view(torch.uint8) != snapshot[0]).any(-1).any(-1).cpu()
    mine = torch.zeros_like(changed)
    for page, row in cache.place[0] + (cache.place[1][63:] if what == "beyond the slots" else []):
        mine[page, row] = True
    if what == "beyond the slots":                        # the tokens that have none do not count for the block's scale
        for page, row in cache.place[1][48:63]:
            mine[page, row] = True
        check(cache, before[1], "k", 1, 63, k[1, :1].double(), 64)
    assert not (changed & ~mine).any()


def test_graph_with_changing_lengths():
    gen = torch.Generator().manual_seed(7)
    cache = Cache8(8, 3, 64, 2, 16)
    k, v = randn(gen, 3, 1, 2, 128).cuda(), randn(gen, 3, 1, 2, 128).cuda()
    lens = torch.tensor([0, 5, 15], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, **cache.more())
        lens.add_(1)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        before = [held(cache, "k", b, 64) for b in range(3)]
        k.copy_(randn(gen, 3, 1, 2, 128) * 2.0**step)
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate((0, 5, 15)):
            check(cache, before[b], "k", b, n + step, k[b].double().cpu(), 64)
