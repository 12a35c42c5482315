"""Performance cases of the cache operators: positions, cache writes, drafted trees, attention weights, eviction.

A case is one pass of one of five kinds, all bf16 with head dimension 128:

    rotary   ``autograd.rotary``: q and k turned by positions of several axes; with ``train`` its gradients too
    append   ``min_fa3_op.append_cache``: new k and v into a cache, q and k turned on the way where the case has a layout
    tree     ``min_fa3_op.forward_tree``: drafted tokens (one token: plain decoding) against a cache
    weights  ``min_fa3_op.cache_weights``: what attention each cache slot received, added up
    evict    ``min_fa3_op.evict_cache``: the slots that received least leave the cache

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

# (query heads, key/value heads): those of the benchmark configurations and tests, and two groups that are no power of two.
HEADS = [(32, 8), (16, 4), (64, 8), (32, 32), (8, 2), (8, 1), (40, 8), (28, 4)]

# How the 64 pairs of a head are shared out among the axes: sections, base, whether each axis starts its frequencies anew,
# whether a pair is two neighbours (or a dimension of the lower and one of the upper half).
LAYOUTS = {
    "text": dict(sections=(64,), base=1e6, restart=False, adjacent=False),
    "text_half": dict(sections=(32,), base=1e4, restart=False, adjacent=True),       # 64 of the 128 dimensions
    "mixed": dict(sections=(16, 24, 24), base=1e6, restart=False, adjacent=False),   # time, height, width in a text model
    "image": dict(sections=(32, 32), base=1e4, restart=True, adjacent=False),
    "video": dict(sections=(22, 21, 21), base=1e4, restart=True, adjacent=True),
}


def listed():
    return [
        # A vision tower's training step: 8 images of 32 x 32 patches, forward and backward.
        dict(name="rotary_image", op="rotary", batch=8, seq=1024, qh=16, kvh=16, layout="image", fused=False, train=True),
        # A clip's tokens on their way into attention, q and k still slices of the fused projection.
        dict(name="rotary_video", op="rotary", batch=1, seq=32760, qh=32, kvh=8, layout="video", fused=True, train=False),
        # One new token for each of 16 sequences: what one call costs.
        dict(name="append_token", op="append", seqs=16, new=1, ragged=False, qh=32, kvh=8, page=64, longest=4000,
             layout="mixed", mix=1),
        # The next chunks of four prompts of different lengths.
        dict(name="append_chunk", op="append", seqs=4, new=2048, ragged=True, qh=32, kvh=8, page=16, longest=8000,
             layout="text", mix=2),
        # A short conversation with a few drafted tokens: what one call costs.
        dict(name="tree_small", op="tree", seqs=1, new=8, ragged=False, tree=True, qh=32, kvh=8, page=16, longest=700, mix=3),
        # Plain decoding: one token for each of 16 sequences.
        dict(name="tree_token", op="tree", seqs=16, new=1, ragged=False, tree=False, qh=32, kvh=8, page=64, longest=8001,
             mix=4),
        # Drafted trees of different sizes.
        dict(name="tree_draft", op="tree", seqs=16, new=32, ragged=True, tree=True, qh=32, kvh=8, page=16, longest=8000,
             mix=5),
        # Large trees, many query heads, long sequences in a cache of one piece each.
        dict(name="tree_wide", op="tree", seqs=8, new=64, ragged=False, tree=True, qh=64, kvh=8, page=0, longest=16000, mix=6),
        # The weights of a decoding step.
        dict(name="weights_token", op="weights", seqs=16, new=1, ragged=False, tree=False, qh=32, kvh=8, page=64,
             longest=8001, mix=7),
        # The weights that a prompt's last 256 tokens give its others.
        dict(name="weights_prompt", op="weights", seqs=2, new=256, ragged=False, tree=False, qh=32, kvh=8, page=16,
             longest=16000, mix=8),
        # One slot leaves each sequence that has outgrown its budget.
        dict(name="evict_step", op="evict", seqs=16, longest=4097, budget=4096, recent=64, kvh=8, page=64, mix=9),
        # Prompts are cut down to their budget.
        dict(name="evict_prompt", op="evict", seqs=8, longest=16000, budget=4000, recent=250, kvh=8, page=16, mix=10),
    ]


def _log_uniform(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    most = {"bytes": max(work(c)["bytes"] for c in listed()), "flops": max(work(c)["flops"] for c in listed())}
    while True:
        op = rng.choice(["rotary", "append", "tree", "tree", "weights", "evict"])
        qh, kvh = rng.choice(HEADS)
        case = dict(op=op)
        if op == "rotary":
            seq = _log_uniform(rng, 1, 32768)
            case.update(batch=_log_uniform(rng, 1, max(1, min(16, 32768 // seq))), seq=seq, qh=qh, kvh=kvh,
                        layout=rng.choice(list(LAYOUTS)), fused=rng.random() < 0.5, train=rng.random() < 0.5)
        elif op == "evict":
            longest = _log_uniform(rng, 100, 32768)
            budget = max(1, round(longest * rng.uniform(0.2, 1.0)))
            case.update(seqs=_log_uniform(rng, 1, max(1, min(32, 131072 // longest))), longest=longest, budget=budget,
                        recent=round(budget * rng.uniform(0, 0.3)), kvh=kvh, page=rng.choice([0, 16, 48, 64, 128]))
        else:
            longest = _log_uniform(rng, 64, 32768)
            new = _log_uniform(rng, 1, {"append": 2048, "tree": 160, "weights": 256}[op])
            case.update(seqs=_log_uniform(rng, 1, max(1, min(64, 131072 // longest))), new=new, ragged=rng.random() < 0.5,
                        qh=qh, kvh=kvh, page=rng.choice([0, 16, 16, 48, 64, 128, 256]), longest=longest)
            if op == "append":
                case["layout"] = rng.choice(["", *LAYOUTS])
            else:
                case["tree"] = new > 1 and rng.random() < 0.7
        if op != "rotary":
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
    if case["op"] == "evict" and longest - case["budget"] == 1:   # a step: every sequence is one over
        return [longest] * case["seqs"]
    return [longest] + [rng.randint(max(1, longest // 4), longest) for _ in range(case["seqs"] - 1)]


def _counts(case):
    """New tokens of each sequence."""
    rng = random.Random(case["mix"] + 1000)
    new = case["new"]
    if not case["ragged"]:
        return [new] * case["seqs"]
    return [rng.randint(max(1, new // 4), new) for _ in range(case["seqs"])]


def work(case):
    row = HEAD_DIM * 2
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        axes = len(LAYOUTS[case["layout"]]["sections"])
        values = tokens * (case["qh"] + case["kvh"]) * HEAD_DIM
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (4 * values) + 8 * axes * tokens, "flops": passes * 3 * values}
    lens = _lengths(case)
    if case["op"] == "evict":
        # Weights in and out, the indices out, and the slots that have to change place: of those kept, the ones behind the
        # budget.  What share of them is kept depends on the weights; here the kept ones lie evenly.
        kvh, moved, slots = case["kvh"], 0, 0
        for n in lens:
            slots += n
            if n > case["budget"]:
                behind = n - case["budget"]
                moved += min(case["recent"], behind) + max(0, behind - case["recent"]) * (case["budget"] - case["recent"]) // n
        return {"bytes": kvh * (slots * 4 + case["seqs"] * (_capacity(case) + case["budget"]) * 4 + moved * 4 * row), "flops": 0}
    counts = _counts(case)
    new, qh, kvh = sum(counts), case["qh"], case["kvh"]
    if case["op"] == "append":
        moved = 4 * new * kvh * row
        flops = 0
        if case["layout"]:
            moved += 2 * new * qh * row + 8 * new * len(LAYOUTS[case["layout"]]["sections"])
            flops = 3 * new * (qh + kvh) * HEAD_DIM
        return {"bytes": moved, "flops": flops}
    slots = sum(n + c for n, c in zip(lens, counts))
    pairs = sum(c * n + c * (c + 1) // 2 for n, c in zip(lens, counts))
    masks = sum(c * c for c in counts) if case["tree"] else 0
    if case["op"] == "tree":
        return {"bytes": 2 * slots * kvh * row + 2 * new * qh * row + 4 * new * qh + masks, "flops": 4 * HEAD_DIM * qh * pairs}
    return {"bytes": slots * kvh * (row + 8) + new * qh * (row + 4) + masks, "flops": 2 * HEAD_DIM * qh * pairs}


def _capacity(case):
    """Slots that a sequence's row of the cache (or of the page table) has."""
    most = case["longest"] + case.get("new", 0)
    return most if case["page"] == 0 else -(-most // case["page"]) * case["page"]


# --------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------
class _State:
    pass


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(torch.bfloat16)


def _frequencies(layout):
    """Frequency and axis of each pair."""
    d = LAYOUTS[layout]
    pairs = sum(d["sections"])
    freq, axis = [], []
    for a, n in enumerate(d["sections"]):
        for j in range(n):
            freq.append(d["base"] ** (-(j / n if d["restart"] else len(freq) / pairs)))
            axis.append(a)
    return freq, axis


def _layout(s, layout):
    freq, axis = _frequencies(layout)
    s.adjacent = LAYOUTS[layout]["adjacent"]
    s.freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    s.axis = torch.tensor(axis, device="cuda")
    if own:
        from min_fa3_demo_b200 import min_fa3_op
        s.axes = min_fa3_op.RotaryAxes(freq, axis, adjacent=s.adjacent)


def _positions(layout, tokens, first):
    """[axes, tokens]: text counts on from ``first``; images and clips have their rows and columns, frames the time."""
    at = torch.arange(tokens, device="cuda") + first
    if layout == "image":
        return torch.stack([at // 32 % 32, at % 32])
    if layout == "video":
        return torch.stack([at // 1560, at // 52 % 30, at % 52])
    if layout == "mixed":                                # every other 64 tokens are an 8 x 8 picture
        seen = at // 64 % 2 == 1
        return torch.stack([at, torch.where(seen, at - at % 64 + at // 8 % 8, at), torch.where(seen, at - at % 64 + at % 8, at)])
    return at[None]


def _trees(case, counts, seed):
    """For each sequence the ancestors (and itself) of every drafted token, [tokens, most tokens], and the same with the
    sequences one behind the other."""
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


def _cache(s, case, gen, used):
    """k_cache, v_cache and, for pages, the block table.  What lies behind a sequence is left over from earlier ones."""
    kvh, page, seqs = case["kvh"], case["page"], case["seqs"]
    cap = _capacity(case)
    if page == 0:
        s.k_cache, s.v_cache, s.table = _normal(gen, seqs, cap, kvh, HEAD_DIM), _normal(gen, seqs, cap, kvh, HEAD_DIM), None
        rows = torch.arange(seqs * cap, device="cuda").view(seqs, cap)
    else:
        need = [-(-n // page) for n in used]
        pool = _normal(gen, sum(need) + 3, 2, page, kvh, HEAD_DIM)          # k and v of a page side by side
        s.k_cache, s.v_cache = pool[:, 0], pool[:, 1]
        order = torch.randperm(sum(need) + 3, device="cuda", generator=gen, dtype=torch.int32)
        s.table = torch.full((seqs, cap // page), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(need):
            s.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
        rows = (s.table.long().clamp(min=0)[:, :, None] * page + torch.arange(page, device="cuda")).view(seqs, cap)
    s.rows = rows                                        # for the plain forms: row of each slot in the cache seen as a list


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
        first = 0 if case["layout"] in ("image", "video") else random.Random(seed).randrange(1 << 20)
        s.positions = _positions(case["layout"], b * n, first).view(-1, b, n)
        s.grads = None
        if case["train"]:
            s.grads = _normal(gen, b, n, qh, HEAD_DIM), _normal(gen, b, n, kvh, HEAD_DIM)
            s.q.requires_grad_(True)
            s.k.requires_grad_(True)
        return s
    s.lens = _lengths(case)
    s.cache_lens = torch.tensor(s.lens, dtype=torch.int32, device="cuda")
    if s.op == "evict":
        _cache(s, case, gen, s.lens)
        # Most slots received little, a few much, some nothing at all.
        w = torch.empty(case["seqs"], case["kvh"], _capacity(case), device="cuda").exponential_(generator=gen) ** 3
        s.weights = torch.where(torch.rand(w.shape, device="cuda", generator=gen) < 0.05, torch.zeros_like(w), w)
        return s
    s.counts = _counts(case)
    total, most = sum(s.counts), max(s.counts)
    s.most = most
    _cache(s, case, gen, [n + c for n, c in zip(s.lens, s.counts)])
    shape = (total,) if case["ragged"] else (case["seqs"], most)
    s.q = _normal(gen, *shape, case["qh"], HEAD_DIM)
    starts = torch.tensor([0] + s.counts).cumsum(0)
    s.cu = starts.to(torch.int32).cuda() if case["ragged"] else None
    # For the plain forms: sequence and number of each row.
    s.seq_of = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(s.counts)).cuda()
    s.num_of = torch.arange(total, device="cuda") - starts.cuda()[s.seq_of]
    if s.op == "append":
        s.k, s.v = _normal(gen, *shape, case["kvh"], HEAD_DIM), _normal(gen, *shape, case["kvh"], HEAD_DIM)
        s.positions = None
        if case["layout"]:
            _layout(s, case["layout"])
            s.positions = torch.cat([_positions(case["layout"], c, n) for n, c in zip(s.lens, s.counts)], 1)
            s.positions = s.positions.view(-1, *shape)
        return s
    s.masks, s.tree_mask = None, None
    if case["tree"]:
        s.masks = _trees(case, s.counts, seed)
        s.tree_mask = torch.cat([s.masks[b, :c] for b, c in enumerate(s.counts)]) if case["ragged"] else s.masks
    if s.op == "weights":
        s.lse = _plain_tree(s)[1]
        s.weights = torch.empty(case["seqs"], case["kvh"], _capacity(case), device="cuda").exponential_(generator=gen)
    return s


# --------------------------------------------------------------------------------------
# Plain forms
# --------------------------------------------------------------------------------------
def _turn(x, cos, sin, adjacent):
    """x [..., heads, 128] by angles [..., pairs]."""
    pairs = cos.size(-1)
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    turned, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    if adjacent:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([out.to(x.dtype), rest], -1)


def _cos_sin(s):
    # Far positions times a frequency need 64 bits.
    angle = s.positions[s.axis].movedim(0, -1).double() * s.freq
    return angle.cos().float(), angle.sin().float()


def _rows_of(cache):
    """The cache's slots as one list [slots, heads, 128]; pages of a pool that holds k and v in turn are not one piece."""
    return cache.reshape(-1, *cache.shape[2:])


def _plain_append(s):
    q, k = s.q, s.k
    if s.positions is not None:
        cos, sin = _cos_sin(s)
        q, k = _turn(q, cos, sin, s.adjacent), _turn(k, cos, sin, s.adjacent)
    slot = s.cache_lens[s.seq_of].long() + s.num_of
    row = s.rows[s.seq_of, slot]
    size = s.k_cache.size(1)
    s.k_cache[row // size, row % size] = k.flatten(0, -3)
    s.v_cache[row // size, row % size] = s.v.flatten(0, -3)
    return (s.k_cache, s.v_cache) if s.positions is None else (q, s.k_cache, s.v_cache)


def _scores(s):
    """Scores of the padded rows [seqs, KVH, group * most, slots], hidden ones -inf, and the slots' rows."""
    seqs, kvh, most = len(s.lens), s.k_cache.size(2), s.most
    qh = s.q.size(-2)
    slots = max(n + c for n, c in zip(s.lens, s.counts))
    q = torch.zeros(seqs, most, qh, HEAD_DIM, device="cuda")
    q[s.seq_of, s.num_of] = s.q.flatten(0, -3).float()
    q = q.view(seqs, most, kvh, qh // kvh, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, -1, HEAD_DIM)
    rows = s.rows[:, :slots]
    k = _rows_of(s.k_cache)[rows].float().permute(0, 2, 3, 1)
    scores = torch.matmul(q, k).mul_(SCALE).view(seqs, kvh, qh // kvh, most, slots)
    drafted = torch.arange(slots, device="cuda") - s.cache_lens[:, None]                       # number among the new ones
    if s.masks is None:
        seen = drafted[:, None, :] <= torch.arange(most, device="cuda")[:, None]
    else:
        inside = ((drafted >= 0) & (drafted < most))[:, None, :]
        index = drafted.clamp(0, most - 1).long()[:, None, :].expand(-1, most, -1)
        seen = (drafted < 0)[:, None, :] | (inside & torch.gather(s.masks, 2, index))
    return scores.masked_fill_(~seen[:, None, None], -math.inf), rows


def _plain_tree(s):
    scores, rows = _scores(s)
    seqs, kvh, group, most, slots = scores.shape
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    # Slots behind a sequence hold what earlier ones left there.
    v = _rows_of(s.v_cache)[rows].float().permute(0, 2, 1, 3)
    out = torch.matmul(p.view(seqs, kvh, group * most, slots), v).view(seqs, kvh, group, most, HEAD_DIM) / total
    lse = (top + total.log()).squeeze(-1).view(seqs, kvh * group, most)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, kvh * group, HEAD_DIM)[s.seq_of, s.num_of].to(torch.bfloat16)
    return out.view(s.q.shape), lse if s.cu is None else lse[s.seq_of, :, s.num_of].T.contiguous()


def _plain_weights(s):
    scores, _ = _scores(s)
    seqs, kvh, group, most, slots = scores.shape
    lse = torch.full((seqs, kvh * group, most), math.inf, device="cuda")
    if s.cu is None:
        lse.copy_(s.lse)
    else:
        lse[s.seq_of, :, s.num_of] = s.lse.T
    p = scores.sub_(lse.view(seqs, kvh, group, most, 1)).exp_()
    s.weights[:, :, :slots] += p.sum((2, 3))
    return s.weights


def _plain_evict(s):
    budget, recent = s.case["budget"], s.case["recent"]
    cap = s.weights.size(2)
    at = torch.arange(cap, device="cuda")
    lens = s.cache_lens.long()[:, None, None]
    kept_lens = lens.clamp(max=budget)
    over = lens > budget
    old = kept_lens - recent                                       # slots for the heaviest
    candidate = at < lens - recent
    value = torch.where(candidate, s.weights, -math.inf)
    order = value.sort(dim=2, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, at.expand_as(order))
    keep = candidate & (rank < old)
    # The i-th kept slot behind the heaviest's place goes to the i-th slot there that is not kept.
    hole, mover = ~keep & (at < old), keep & (at >= old)
    where_hole = torch.where(hole, hole.cumsum(2) - 1, cap)
    movers = torch.full((*keep.shape[:2], cap + 1), 0, device="cuda")
    movers.scatter_(2, torch.where(mover, mover.cumsum(2) - 1, cap), at.expand_as(keep))
    index = torch.where(hole, torch.gather(movers, 2, where_hole), at.expand_as(keep))
    index = torch.where(at >= old, at + (lens - kept_lens), index)  # the last ones, in their order
    index = torch.where(over, index, at)
    index = torch.where(at < kept_lens, index, -1)
    source = index.clamp(min=0)
    weights = torch.where(index >= 0, torch.gather(s.weights, 2, source), 0.0)
    size, heads = s.k_cache.size(1), torch.arange(s.weights.size(1), device="cuda")[:, None]
    seq = torch.arange(len(s.lens), device="cuda")[:, None, None]
    to, come = s.rows[:, None, :budget].expand(-1, heads.size(0), -1), s.rows[seq, source[:, :, :budget]]
    come = torch.where(index[:, :, :budget] >= 0, come, to)
    for cache in (s.k_cache, s.v_cache):
        cache[to // size, to % size, heads] = cache[come // size, come % size, heads]
    return kept_lens.view(-1).to(torch.int32), weights, index[:, :, :budget].to(torch.int32), s.k_cache, s.v_cache


def _plain_rotary(s):
    q, k = s.q.detach(), s.k.detach()
    cos, sin = _cos_sin(s)
    out = _turn(q, cos, sin, s.adjacent), _turn(k, cos, sin, s.adjacent)
    if s.grads is None:
        return out
    return (*out, _turn(s.grads[0], cos, -sin, s.adjacent), _turn(s.grads[1], cos, -sin, s.adjacent))


def run(s):
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "tree": _plain_tree, "weights": _plain_weights,
                "evict": _plain_evict}[s.op](s)
    from min_fa3_demo_b200 import autograd, min_fa3_op
    if s.op == "rotary":
        out = autograd.rotary(s.q, s.k, s.positions, s.axes)
        return out if s.grads is None else (*out, *torch.autograd.grad(out, (s.q, s.k), s.grads))
    if s.op == "append":
        if s.positions is None:
            min_fa3_op.append_cache(s.k, s.v, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens=s.cu)
            return s.k_cache, s.v_cache
        q = min_fa3_op.append_cache(s.k, s.v, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens=s.cu,
                                    q=s.q, positions=s.positions, axes=s.axes)
        return q, s.k_cache, s.v_cache
    if s.op == "tree":
        return min_fa3_op.forward_tree(s.q, s.k_cache, s.v_cache, s.cache_lens, block_table=s.table, cu_seqlens_q=s.cu,
                                       max_seqlen_q=s.most, tree_mask=s.tree_mask, return_lse=True)
    if s.op == "weights":
        return min_fa3_op.cache_weights(s.q, s.lse, s.k_cache, s.cache_lens, s.weights, block_table=s.table,
                                        cu_seqlens_q=s.cu, max_seqlen_q=s.most, tree_mask=s.tree_mask)
    lens, weights, index = min_fa3_op.evict_cache(s.k_cache, s.v_cache, s.weights, s.cache_lens, s.case["budget"],
                                                  recent=s.case["recent"], block_table=s.table)
    return lens, weights, index, s.k_cache, s.v_cache


# --------------------------------------------------------------------------------------
# The same in 64 bits, token by token, sequence by sequence or head by head
# --------------------------------------------------------------------------------------
def _exact_turn(x, positions, layout, sign):
    """x [tokens, heads, 128] as complex numbers times exp(i angle)."""
    freq, axis = _frequencies(layout)
    pairs = len(freq)
    x = x.double()
    first = torch.arange(pairs, device="cuda") * 2 if LAYOUTS[layout]["adjacent"] else torch.arange(pairs, device="cuda")
    second = first + 1 if LAYOUTS[layout]["adjacent"] else first + pairs
    angle = torch.stack([positions[a].double() * f for f, a in zip(freq, axis)], 1)[:, None]
    z = torch.polar(torch.ones_like(angle), sign * angle) * torch.complex(x[:, :, first], x[:, :, second])
    out = x.clone()
    out[:, :, first], out[:, :, second] = z.real, z.imag
    return out


def _sequences(s):
    """(sequence, first row, rows, its slots' rows) of each sequence."""
    first = 0
    for b, (n, c) in enumerate(zip(s.lens, s.counts)):
        yield b, first, c, s.rows[b, :n + c]
        first += c


def _exact_scores(s, b, c, q, k, n):
    """Scores [heads, rows, slots] of one sequence."""
    group = q.size(1) // k.size(1)
    score = torch.einsum("thd,shd->hts", q.double(), k.double().repeat_interleave(group, 1)) / math.sqrt(HEAD_DIM)
    seen = torch.ones(c, n + c, dtype=torch.bool, device="cuda")
    seen[:, n:] = torch.ones(c, c, dtype=torch.bool, device="cuda").tril() if s.masks is None else s.masks[b, :c, :c]
    return torch.where(seen, score, -math.inf)


def _exact_evict(s):
    budget, recent = s.case["budget"], s.case["recent"]
    w = s.weights.double().cpu().numpy()
    seqs, kvh, cap = w.shape
    weights, index = np.zeros_like(w), np.full((seqs, kvh, budget), -1)
    for b, n in enumerate(s.lens):
        m = min(n, budget)
        for h in range(kvh):
            place = list(range(m))
            if n > budget:
                best = sorted(range(n - recent), key=lambda j: (-w[b, h, j], j))[:m - recent]
                late = iter(sorted(j for j in best if j >= m - recent))
                stay = {j for j in best if j < m - recent}
                place = [j if j in stay else next(late) for j in range(m - recent)] + list(range(n - recent, n))
            index[b, h, :m] = place
            weights[b, h, :m] = w[b, h, place]
    index = torch.from_numpy(index).cuda()
    lens = torch.tensor([min(n, budget) for n in s.lens])
    caches = []
    for cache in (s.k_cache, s.v_cache):
        flat = _rows_of(cache).clone()
        new = flat.clone()
        for b, n in enumerate(lens.tolist()):
            for h in range(kvh):
                new[s.rows[b, :n], h] = flat[s.rows[b, index[b, h, :n]], h]
        caches.append(new.view(cache.shape))
    return lens, torch.from_numpy(weights), index, *caches


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "rotary":
        flat = s.positions.flatten(1)
        outs = [_exact_turn(x.detach().flatten(0, 1), flat, case["layout"], sign).view(x.shape)
                for x, sign in [(s.q, 1), (s.k, 1)] + ([(s.grads[0], -1), (s.grads[1], -1)] if case["train"] else [])]
        return tuple(outs)
    if s.op == "evict":
        return _exact_evict(s)
    q = s.q.flatten(0, -3)
    if s.op == "append":
        k, v, caches = s.k.flatten(0, -3).double(), s.v.flatten(0, -3), []
        if case["layout"]:
            flat = s.positions.flatten(1)
            q, k = (_exact_turn(x, flat, case["layout"], 1) for x in (q, k))
        for cache, new in ((s.k_cache, k), (s.v_cache, v.double())):
            flat = _rows_of(cache).double()
            for b, first, c, rows in _sequences(s):
                flat[rows[s.lens[b]:]] = new[first:first + c]
            caches.append(flat.view(cache.shape))
        return (*caches,) if not case["layout"] else (q.view(s.q.shape), *caches)
    if work(case)["flops"] > 2e12:                       # more than about 20 seconds in 64 bits
        return None
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.size(1), q.size(0), device="cuda").double()
    weights = s.weights.double() if s.op == "weights" else None
    for b, first, c, rows in _sequences(s):
        n = s.lens[b]
        score = _exact_scores(s, b, c, q[first:first + c], _rows_of(s.k_cache)[rows], n)
        if s.op == "weights":
            given = s.lse[b] if s.cu is None else s.lse[:, first:first + c]
            p = (score - given.double()[:, :, None]).exp()
            weights[b, :, :n + c] += p.view(s.k_cache.size(2), -1, c, n + c).sum((1, 2))
            continue
        p = score.softmax(2)
        v = _rows_of(s.v_cache)[rows].double().repeat_interleave(q.size(1) // s.k_cache.size(2), 1)
        out[first:first + c] = torch.einsum("hts,shd->thd", p, v)
        lse[:, first:first + c] = score.logsumexp(2)
    if s.op == "weights":
        return weights
    return out.view(s.q.shape), lse if s.cu is not None else lse.view(q.size(1), case["seqs"], -1).transpose(0, 1)
