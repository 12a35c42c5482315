"""Performance cases of the 8-bit cache and of stretched rotary positions.

A case is one pass of one of three kinds, with head dimension 128:

    rotary   ``autograd.rotary``: q and k turned by positions stretched beyond the length a model was trained on; with ``train``
             their gradients too
    append   ``min_fa3_op.append_cache``: new k and v into a cache of float8_e4m3fn with a scale for each block of slots and K/V
             head, q and k turned on the way where the case has a layout
    tree     ``min_fa3_op.forward_tree``: drafted tokens, the next token or a prompt's next chunk against such a cache

``own`` chooses what ``run()`` does: the library's calls, or the same operators in elementary torch operations.
``listed()`` gives the cases, ``draw()`` more of the same ranges, ``prepare()`` / ``run()`` execute one, ``work()``
counts the bytes and operations it cannot do without, ``exact()`` gives the result in 64 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

HEAD_DIM = 128
SCALE = 1.0 / math.sqrt(HEAD_DIM)
MOST8 = 448.0                  # largest e4m3 value
E4M3 = torch.float8_e4m3fn

# (query heads, key/value heads): those of the benchmark configurations and tests, and two groups that are no power of two.
HEADS = [(32, 8), (16, 4), (64, 8), (32, 32), (8, 2), (8, 1), (40, 8), (28, 4)]

# How many pairs of a head turn, with which base, whether a pair is two neighbours (or a dimension of the lower and one of the
# upper half), and how they are stretched: factor, length trained on, and between how many turns in that length the
# pairs go over from the stretched frequency to their own; what the turned pairs are multiplied by.
LAYOUTS = {
    "long": dict(pairs=64, base=1e6, adjacent=False, factor=4.0, length=32768, slow=1.0, fast=32.0, magnitude=0.1 * math.log(4.0) + 1),
    "long_part": dict(pairs=32, base=1e4, adjacent=True, factor=16.0, length=4096, slow=1.0, fast=32.0, magnitude=0.1 * math.log(16.0) + 1),
    "smooth": dict(pairs=64, base=5e5, adjacent=False, factor=8.0, length=8192, slow=1.0, fast=4.0, magnitude=1.0),
}


def listed():
    return [
        # A training step at a longer context than before: forward and backward.
        dict(name="rotary_long_train", op="rotary", batch=2, seq=8192, qh=32, kvh=8, layout="long", fused=False, train=True),
        # A long prompt on its way into attention, q and k still slices of the fused projection.
        dict(name="rotary_long_prompt", op="rotary", batch=1, seq=30001, qh=32, kvh=8, layout="long_part", fused=True, train=False),
        # One new token for each of 16 sequences: what one call costs.
        dict(name="append8_token", op="append", seqs=16, new=1, ragged=False, qh=32, kvh=8, page=64, block=16, longest=4000,
             layout="long", mix=1),
        # Drafted tokens, which begin inside of blocks.
        dict(name="append8_draft", op="append", seqs=32, new=24, ragged=True, qh=32, kvh=8, page=64, block=32, longest=4000,
             layout="smooth", mix=2),
        # The next chunks of four prompts of different lengths.
        dict(name="append8_chunk", op="append", seqs=4, new=2048, ragged=True, qh=32, kvh=8, page=16, block=16, longest=8000,
             layout="long", mix=3),
        # A short conversation with a few drafted tokens: what one call costs.
        dict(name="tree8_small", op="tree", seqs=1, new=8, ragged=False, tree=True, qh=32, kvh=8, page=16, block=16, longest=700, mix=4),
        # Plain decoding: one token for each of 16 sequences.
        dict(name="tree8_token", op="tree", seqs=16, new=1, ragged=False, tree=False, qh=32, kvh=8, page=64, block=16, longest=8001,
             mix=5),
        # One token against a single long context.
        dict(name="tree8_long", op="tree", seqs=1, new=1, ragged=False, tree=False, qh=32, kvh=8, page=64, block=64, longest=131072, mix=6),
        # Drafted trees of different sizes.
        dict(name="tree8_draft", op="tree", seqs=16, new=32, ragged=True, tree=True, qh=32, kvh=8, page=16, block=16, longest=8000,
             mix=7),
        # Large trees, many query heads, long sequences in a cache of one piece each.
        dict(name="tree8_wide", op="tree", seqs=8, new=64, ragged=False, tree=True, qh=64, kvh=8, page=0, block=32, longest=16000, mix=8),
        # The next chunks of two prompts against what the cache holds of them.
        dict(name="tree8_chunk", op="tree", seqs=2, new=1000, ragged=False, tree=False, qh=32, kvh=8, page=64, block=64, longest=8000,
             mix=9),
    ]


def _log_uniform(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    most = {"bytes": max(work(c)["bytes"] for c in listed()), "flops": max(work(c)["flops"] for c in listed())}
    while True:
        op = rng.choice(["rotary", "append", "append", "tree", "tree", "tree"])
        qh, kvh = rng.choice(HEADS)
        case = dict(op=op)
        if op == "rotary":
            seq = _log_uniform(rng, 1, 32768)
            case.update(batch=_log_uniform(rng, 1, max(1, min(16, 32768 // seq))), seq=seq, qh=qh, kvh=kvh,
                        layout=rng.choice(list(LAYOUTS)), fused=rng.random() < 0.5, train=rng.random() < 0.5)
        else:
            longest = _log_uniform(rng, 64, 131072)
            new = _log_uniform(rng, 1, {"append": 2048, "tree": 1000}[op])
            page = rng.choice([0, 16, 48, 64, 128, 256])
            block = rng.choice([b for b in (16, 32, 64, 128) if page % b == 0])
            case.update(seqs=_log_uniform(rng, 1, max(1, min(64, 131072 // longest))), new=new, ragged=rng.random() < 0.5,
                        qh=qh, kvh=kvh, page=page, block=block, longest=longest)
            if op == "append":
                case["layout"] = rng.choice(["", *LAYOUTS])
            else:
                case["tree"] = 1 < new <= 160 and rng.random() < 0.7
            case["mix"] = rng.randrange(1000)
        w = work(case)
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return case


# --------------------------------------------------------------------------------------
# Sizes
# --------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens in the cache of each sequence: the longest, and others down to a quarter of it."""
    rng = random.Random(case["mix"])
    longest = case["longest"]
    return [longest] + [rng.randint(max(1, longest // 4), longest) for _ in range(case["seqs"] - 1)]


def _counts(case):
    """New tokens of each sequence."""
    rng = random.Random(case["mix"] + 1000)
    new = case["new"]
    if not case["ragged"]:
        return [new] * case["seqs"]
    return [rng.randint(max(1, new // 4), new) for _ in range(case["seqs"])]


def _capacity(case):
    """Slots that a sequence's row of the cache (or of the page table) has."""
    most = case["longest"] + case["new"]
    return most if case["page"] == 0 else -(-most // case["page"]) * case["page"]


def work(case):
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["qh"] + case["kvh"]) * HEAD_DIM
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (4 * values) + 8 * tokens, "flops": passes * 4 * values}
    lens, counts = _lengths(case), _counts(case)
    new, qh, kvh, block = sum(counts), case["qh"], case["kvh"], case["block"]
    if case["op"] == "append":
        # k and v in at 16 bits and out at 8, the scales of the blocks that are begun, in and out where they held tokens.
        scales = sum((n + c - 1) // block - n // block + 1 + (n % block > 0) for n, c in zip(lens, counts))
        moved = 2 * new * kvh * HEAD_DIM * 3 + 2 * scales * kvh * 4
        flops = 4 * new * kvh * HEAD_DIM
        if case["layout"]:
            moved += 4 * new * qh * HEAD_DIM + 8 * new
            flops += 4 * new * (qh + kvh) * HEAD_DIM
        return {"bytes": moved, "flops": flops}
    slots = sum(n + c for n, c in zip(lens, counts))
    blocks = sum(-(-(n + c) // block) for n, c in zip(lens, counts))
    pairs = sum(c * n + c * (c + 1) // 2 for n, c in zip(lens, counts))
    masks = sum(c * c for c in counts) if case["tree"] else 0
    return {"bytes": 2 * kvh * (slots * HEAD_DIM + blocks * 4) + 4 * new * qh * HEAD_DIM + 4 * new * qh + masks,
            "flops": 4 * HEAD_DIM * qh * pairs}


# --------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------
class _State:
    pass


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(torch.bfloat16)


def _frequencies(layout):
    """Frequency of each pair before stretching, and after it."""
    d = LAYOUTS[layout]
    plain = [d["base"] ** (-i / d["pairs"]) for i in range(d["pairs"])]
    stretched = []
    for f in plain:
        turns = d["length"] * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - d["slow"]) / (d["fast"] - d["slow"])))
        stretched.append((1 - keep) * f / d["factor"] + keep * f)
    return plain, stretched


def _layout(s, layout):
    d = LAYOUTS[layout]
    plain, stretched = _frequencies(layout)
    s.adjacent, s.magnitude = d["adjacent"], d["magnitude"]
    s.freq = torch.tensor(stretched, dtype=torch.float64, device="cuda")
    if own:
        from min_fa3_demo_b200 import min_fa3_op
        s.axes = min_fa3_op.RotaryAxes(plain, adjacent=d["adjacent"]).stretched(
            d["factor"], d["length"], slow=d["slow"], fast=d["fast"], magnitude=d["magnitude"])


def _trees(counts, seed):
    """For each sequence the ancestors (and itself) of every drafted token, [sequences, tokens, tokens]."""
    rng = random.Random(seed)
    most = max(counts)
    masks = np.zeros((len(counts), most, most), dtype=bool)
    for b, c in enumerate(counts):
        for i in range(c):
            parent = rng.randint(max(-1, i // 2 - 2), i - 1)   # a token has about two children
            if parent >= 0:
                masks[b, i] = masks[b, parent]
            masks[b, i, i] = True
    return torch.from_numpy(masks).cuda()


def _power(most):
    """The smallest power of two that brings ``most`` down to 448, within 2^-64 .. 2^64."""
    mantissa, exponent = torch.frexp(most)               # most = mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > MOST8 / 512).to(exponent.dtype)
    exponent = torch.where(most > 0, exponent, torch.full_like(exponent, -64)).clamp(-64, 64)
    return torch.ldexp(torch.ones_like(most), exponent)


def _filled(gen, pages, size, kvh, block):
    """Pages with random contents, as e4m3 and scales; a token's values have a size of their own, as in a model."""
    blocks = -(-size // block)
    cache = torch.empty(pages, size, kvh, HEAD_DIM, device="cuda", dtype=E4M3)
    scales = torch.empty(pages, blocks, kvh, device="cuda")
    step = max(1, (1 << 26) // (size * kvh * HEAD_DIM))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.zeros(n, blocks * block, kvh, HEAD_DIM, device="cuda")
        x[:, :size] = torch.randn(n, size, kvh, HEAD_DIM, device="cuda", generator=gen)
        x[:, :size] *= torch.randn(n, size, kvh, 1, device="cuda", generator=gen).mul_(0.4).exp_()
        x = x.view(n, blocks, block, kvh, HEAD_DIM)
        s = _power(x.abs().amax((2, 4)))
        scales[at:at + n] = s
        cache[at:at + n] = (x / s[:, :, None, :, None]).view(n, blocks * block, kvh, HEAD_DIM)[:, :size].to(E4M3)
    return cache, scales


def _cache(s, case, gen, used):
    """Caches, scales and, for pages, the block table.  What lies behind a sequence is left over from earlier ones."""
    kvh, page, seqs, block = case["kvh"], case["page"], case["seqs"], case["block"]
    cap = _capacity(case)
    if page == 0:
        s.k_cache, s.k_scales = _filled(gen, seqs, cap, kvh, block)
        s.v_cache, s.v_scales = _filled(gen, seqs, cap, kvh, block)
        s.table = None
        s.rows = torch.arange(seqs * cap, device="cuda").view(seqs, cap)
        row_of = torch.arange(cap, device="cuda")
        s.scale_rows = torch.arange(seqs, device="cuda")[:, None] * s.k_scales.size(1) + row_of // block
        return
    need = [-(-n // page) for n in used]
    pages = sum(need) + 3
    pool, scales = _filled(gen, 2 * pages, page, kvh, block)                 # k and v of a page side by side
    pool, scales = pool.view(pages, 2, page, kvh, HEAD_DIM), scales.view(pages, 2, -1, kvh)
    s.k_cache, s.v_cache, s.k_scales, s.v_scales = pool[:, 0], pool[:, 1], scales[:, 0], scales[:, 1]
    order = torch.randperm(pages, device="cuda", generator=gen, dtype=torch.int32)
    s.table = torch.full((seqs, cap // page), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(need):
        s.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
    at = s.table.long().clamp(min=0)[:, :, None]
    row_of = torch.arange(page, device="cuda")
    s.rows = (at * page + row_of).view(seqs, cap)         # for the plain forms: row of each slot in the cache seen as a list,
    s.scale_rows = (at * (page // block) + row_of // block).view(seqs, cap)  # and its scale's in the list of scales


def prepare(case, seed):
    s = _State()
    s.case, s.op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if s.op == "rotary":
        b, n, qh, kvh = case["batch"], case["seq"], case["qh"], case["kvh"]
        if case["fused"]:
            both = _normal(gen, b, n, qh + 2 * kvh, HEAD_DIM)
            s.q, s.k = both[:, :, :qh], both[:, :, qh:qh + kvh]
        else:
            s.q, s.k = _normal(gen, b, n, qh, HEAD_DIM), _normal(gen, b, n, kvh, HEAD_DIM)
        _layout(s, case["layout"])
        first = random.Random(seed).randrange(1 << 17)
        s.positions = (torch.arange(n, device="cuda") + first).expand(1, b, n)
        s.grads = None
        if case["train"]:
            s.grads = _normal(gen, b, n, qh, HEAD_DIM), _normal(gen, b, n, kvh, HEAD_DIM)
            s.q.requires_grad_(True)
            s.k.requires_grad_(True)
        return s
    s.lens, s.counts = _lengths(case), _counts(case)
    s.cache_lens = torch.tensor(s.lens, dtype=torch.int32, device="cuda")
    total, s.most = sum(s.counts), max(s.counts)
    _cache(s, case, gen, [n + c for n, c in zip(s.lens, s.counts)])
    shape = (total,) if case["ragged"] else (case["seqs"], s.most)
    s.q = _normal(gen, *shape, case["qh"], HEAD_DIM)
    starts = torch.tensor([0] + s.counts).cumsum(0)
    s.cu = starts.to(torch.int32).cuda() if case["ragged"] else None
    # For the plain forms: sequence and number of each row.
    s.seq_of = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(s.counts)).cuda()
    s.num_of = torch.arange(total, device="cuda") - starts.cuda()[s.seq_of]
    if s.op == "append":
        s.k, s.v = _normal(gen, *shape, case["kvh"], HEAD_DIM), _normal(gen, *shape, case["kvh"], HEAD_DIM)
        # Now and then a token far larger than those before it, for which a block's scale has to grow.
        for x in (s.k, s.v):
            x *= torch.where(torch.rand(*shape, case["kvh"], 1, device="cuda", generator=gen) < 0.05, 6.0, 1.0).to(torch.bfloat16)
        s.positions = None
        if case["layout"]:
            _layout(s, case["layout"])
            s.positions = (s.cache_lens[s.seq_of].long() + s.num_of).view(1, *shape)
        return s
    s.masks, s.tree_mask = None, None
    if case["tree"]:
        s.masks = _trees(s.counts, seed)
        s.tree_mask = torch.cat([s.masks[b, :c] for b, c in enumerate(s.counts)]) if case["ragged"] else s.masks
    return s


# --------------------------------------------------------------------------------------
# Plain forms
# --------------------------------------------------------------------------------------
def _turn(x, cos, sin, adjacent):
    """x [..., heads, 128] by angles [..., pairs], in 32 bits."""
    pairs = cos.size(-1)
    cos, sin, x = cos.unsqueeze(-2), sin.unsqueeze(-2), x.float()
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if adjacent:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([out, rest], -1)


def _cos_sin(s):
    # Far positions times a frequency need 64 bits.
    angle = s.positions[0].double()[..., None] * s.freq
    return (angle.cos() * s.magnitude).float(), (angle.sin() * s.magnitude).float()


def _plain_rotary(s):
    cos, sin = _cos_sin(s)
    out = [_turn(x.detach(), cos, sin, s.adjacent).to(torch.bfloat16) for x in (s.q, s.k)]
    if s.grads is not None:
        out += [_turn(x, cos, -sin, s.adjacent).to(torch.bfloat16) for x in s.grads]
    return tuple(out)


def _plain_write(s, cache, scales, x):
    """x [tokens, heads, 128] behind what the cache holds; blocks keep their scale while it is large enough."""
    block, heads = s.case["block"], x.size(1)
    lens = s.cache_lens.long()
    slot = lens[s.seq_of] + s.num_of
    # Blocks of a sequence from the one that its first new token falls into, [sequences, blocks].
    first = lens // block
    blocks = (block - 1 + s.most + block - 1) // block
    mine = s.seq_of * blocks + slot // block - first[s.seq_of]
    most = torch.zeros(lens.size(0) * blocks, heads, device="cuda")
    most.scatter_reduce_(0, mine[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    most = most.view(-1, blocks, heads)
    new_tokens = torch.zeros(lens.size(0) * blocks, device="cuda", dtype=torch.bool)
    new_tokens[mine] = True
    # A block's scale: that of its first slot.
    cap = s.rows.size(1)
    begin = ((first[:, None] + torch.arange(blocks, device="cuda")) * block).clamp(max=cap - 1)
    seqs = torch.arange(lens.size(0), device="cuda")
    place = s.scale_rows[seqs[:, None], begin]
    page, number = place // scales.size(1), place % scales.size(1)
    before = scales[page, number]
    held = (begin < lens[:, None])[:, :, None]
    after = torch.where(held & (most <= MOST8 * before), before, _power(most))
    # Tokens that the first block holds already.
    old = (first * block)[:, None] + torch.arange(block, device="cuda")
    is_old, old = old < lens[:, None], old.clamp(max=cap - 1)
    row = s.rows[seqs[:, None], old]
    size = cache.size(1)
    at = row // size, row % size
    now = cache[at].float()
    again = (now * (before[:, 0] / after[:, 0])[:, None, :, None]).to(E4M3)
    keep = is_old & (s.cache_lens > 0)[:, None]
    at = at[0][keep], at[1][keep]
    cache.view(torch.uint8)[at] = again.view(torch.uint8)[keep]
    there = new_tokens.view(-1, blocks)
    scales[page[there], number[there]] = after[there]
    row = s.rows[s.seq_of, slot]
    values = (x / after.view(-1, heads)[mine][:, :, None]).to(E4M3)
    cache.view(torch.uint8)[row // size, row % size] = values.view(torch.uint8)


def _plain_append(s):
    q, k, v = s.q, s.k.float(), s.v.float()
    if s.positions is not None:
        cos, sin = _cos_sin(s)
        q, k = _turn(q, cos, sin, s.adjacent).to(torch.bfloat16), _turn(k, cos, sin, s.adjacent)
    _plain_write(s, s.k_cache, s.k_scales, k.flatten(0, -3))
    _plain_write(s, s.v_cache, s.v_scales, v.flatten(0, -3))
    out = s.k_cache, s.v_cache, s.k_scales, s.v_scales
    return out if s.positions is None else (q, *out)


def _values(s, cache, scales, slots):
    """What the first slots stand for, [sequences, slots, heads, 128] in 32 bits."""
    size, blocks = cache.size(1), scales.size(1)
    row, place = s.rows[:, :slots], s.scale_rows[:, :slots]
    return cache[row // size, row % size].float() * scales[place // blocks, place % blocks][..., None]


def _plain_tree(s):
    seqs, kvh, most, qh = len(s.lens), s.k_cache.size(2), s.most, s.q.size(-2)
    slots = max(n + c for n, c in zip(s.lens, s.counts))
    q = torch.zeros(seqs, most, qh, HEAD_DIM, device="cuda")
    q[s.seq_of, s.num_of] = s.q.flatten(0, -3).float()
    q = q.view(seqs, most, kvh, qh // kvh, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, -1, HEAD_DIM)
    k = _values(s, s.k_cache, s.k_scales, slots).permute(0, 2, 3, 1)
    scores = torch.matmul(q, k).mul_(SCALE).view(seqs, kvh, qh // kvh, most, slots)
    drafted = torch.arange(slots, device="cuda") - s.cache_lens[:, None]                       # number among the new ones
    if s.masks is None:
        seen = drafted[:, None, :] <= torch.arange(most, device="cuda")[:, None]
    else:
        inside = ((drafted >= 0) & (drafted < most))[:, None, :]
        index = drafted.clamp(0, most - 1).long()[:, None, :].expand(-1, most, -1)
        seen = (drafted < 0)[:, None, :] | (inside & torch.gather(s.masks, 2, index))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = _values(s, s.v_cache, s.v_scales, slots).permute(0, 2, 1, 3)
    out = torch.matmul(p.view(seqs, kvh, -1, slots), v).view(seqs, kvh, qh // kvh, most, HEAD_DIM) / total
    lse = (top + total.log()).squeeze(-1).view(seqs, qh, most)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, qh, HEAD_DIM)[s.seq_of, s.num_of].to(torch.bfloat16)
    return out.view(s.q.shape), lse if s.cu is None else lse[s.seq_of, :, s.num_of].T.contiguous()


def run(s):
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "tree": _plain_tree}[s.op](s)
    from min_fa3_demo_b200 import autograd, min_fa3_op
    if s.op == "rotary":
        out = autograd.rotary(s.q, s.k, s.positions, s.axes)
        return out if s.grads is None else (*out, *torch.autograd.grad(out, (s.q, s.k), s.grads))
    if s.op == "append":
        caches = s.k_cache, s.v_cache, s.k_scales, s.v_scales
        if s.positions is None:
            min_fa3_op.append_cache(s.k, s.v, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens=s.cu,
                                    k_scales=s.k_scales, v_scales=s.v_scales)
            return caches
        q = min_fa3_op.append_cache(s.k, s.v, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens=s.cu,
                                    q=s.q, positions=s.positions, axes=s.axes, k_scales=s.k_scales, v_scales=s.v_scales)
        return (q, *caches)
    return min_fa3_op.forward_tree(s.q, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens_q=s.cu,
                                   max_seqlen_q=s.most, tree_mask=s.tree_mask, return_lse=True, k_scales=s.k_scales,
                                   v_scales=s.v_scales)


# --------------------------------------------------------------------------------------
# The same in 64 bits, token by token and sequence by sequence
# --------------------------------------------------------------------------------------
def _exact_turn(x, positions, layout, sign):
    """x [tokens, heads, 128] as complex numbers times magnitude * exp(i angle)."""
    d = LAYOUTS[layout]
    freq = _frequencies(layout)[1]
    pairs = len(freq)
    x = x.double()
    first = torch.arange(pairs, device="cuda") * 2 if d["adjacent"] else torch.arange(pairs, device="cuda")
    second = first + 1 if d["adjacent"] else first + pairs
    angle = torch.stack([positions.double() * f for f in freq], 1)[:, None]
    z = torch.polar(torch.full_like(angle, d["magnitude"]), sign * angle) * torch.complex(x[:, :, first], x[:, :, second])
    out = x.clone()
    out[:, :, first], out[:, :, second] = z.real, z.imag
    return out


def _to_e4m3(x):
    """Values of 64 bits rounded to a multiple of 1/8 of their power of two (2^-9 at least), ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return torch.round(x / step).mul(step).clamp(-448, 448)


def _sequences(s):
    """(sequence, first row, rows) of each sequence."""
    first = 0
    for b, c in enumerate(s.counts):
        yield b, first, c
        first += c


def _exact_write(s, cache, scales, x):
    block, size, blocks = s.case["block"], cache.size(1), scales.size(1)
    cache, scales = cache.double().clone(), scales.double().clone()
    flat, flat_scales = cache.view(-1, *cache.shape[2:]), scales.view(-1, scales.size(2))
    assert flat.size(0) == cache.size(0) * size and flat_scales.size(0) == scales.size(0) * blocks
    for b, first, c in _sequences(s):
        n = s.lens[b]
        for j in range(n // block, (n + c - 1) // block + 1):
            lo, hi = max(n, j * block), min(n + c, (j + 1) * block)
            new = x[first + lo - n:first + hi - n]
            most = new.abs().amax((0, 2))
            place = s.scale_rows[b, j * block]
            scale = torch.exp2(torch.ceil(torch.log2(most / 448).clamp(-64, 64)))
            if lo > j * block:
                had = flat_scales[place]
                scale = torch.where(most <= 448 * had, had, scale)
                rows = s.rows[b, j * block:lo]
                flat[rows] = _to_e4m3(flat[rows] * (had / scale)[None, :, None])
            flat_scales[place] = scale
            flat[s.rows[b, lo:hi]] = _to_e4m3(new / scale[None, :, None])
    return cache, scales


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "rotary":
        flat = s.positions[0].flatten()
        outs = [_exact_turn(x.detach().flatten(0, 1), flat, case["layout"], sign).view(x.shape)
                for x, sign in [(s.q, 1), (s.k, 1)] + ([(s.grads[0], -1), (s.grads[1], -1)] if case["train"] else [])]
        return tuple(outs)
    q = s.q.flatten(0, -3)
    if s.op == "append":
        k, v = s.k.flatten(0, -3).double(), s.v.flatten(0, -3).double()
        if case["layout"]:
            q, k = (_exact_turn(x, s.positions.flatten(), case["layout"], 1) for x in (q, k))
        k_cache, k_scales = _exact_write(s, s.k_cache, s.k_scales, k)
        v_cache, v_scales = _exact_write(s, s.v_cache, s.v_scales, v)
        out = k_cache, v_cache, k_scales, v_scales
        return out if not case["layout"] else (q.view(s.q.shape), *out)
    if work(case)["flops"] > 2e12:                       # more than about 20 seconds in 64 bits
        return None
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.size(1), q.size(0), device="cuda").double()
    heads, kvh = q.size(1), s.k_cache.size(2)
    for b, first, c in _sequences(s):
        n = s.lens[b]
        row, place = s.rows[b, :n + c], s.scale_rows[b, :n + c]
        size, blocks = s.k_cache.size(1), s.k_scales.size(1)
        k, v = (cache[row // size, row % size].double() * scales[place // blocks, place % blocks].double()[..., None]
                for cache, scales in ((s.k_cache, s.k_scales), (s.v_cache, s.v_scales)))
        seen = torch.ones(c, n + c, dtype=torch.bool, device="cuda")
        seen[:, n:] = torch.ones(c, c, dtype=torch.bool, device="cuda").tril() if s.masks is None else s.masks[b, :c, :c]
        for h in range(heads):
            g = h // (heads // kvh)
            score = q[first:first + c, h].double() @ k[:, g].T / math.sqrt(HEAD_DIM)
            score = torch.where(seen, score, -math.inf)
            out[first:first + c, h] = score.softmax(1) @ v[:, g]
            lse[h, first:first + c] = score.logsumexp(1)
    return out.view(s.q.shape), lse if s.cu is not None else lse.view(heads, case["seqs"], -1).transpose(0, 1)
