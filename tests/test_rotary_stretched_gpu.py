"""Stretched rotary axes on the GPU against the formula in 64 bits: rotary, its gradients, and writes of caches in bf16.

Tolerance: that of the tests of ``rotary`` times the magnitude: one rounding to bf16, and a few in 32 bits, one more for the
magnitude's product with sine and cosine."""
from __future__ import annotations

import math

import pytest
import torch

import min_fa3_op
from cache_util import BF16_HALF_STEP, Cache, randn, turn
from min_fa3_demo_b200 import autograd

pytestmark = pytest.mark.gpu

# Sections, base, adjacent; factor, trained length, slow, fast, magnitude.
CASES = {
    "long": ((64,), 1e6, False, 4, 32768, 1, 32, None),
    "smooth": ((64,), 5e5, False, 8, 8192, 1, 4, 1.0),
    "linear": ((32,), 1e4, True, 2, 4096, math.inf, math.inf, 1.0),
    "axes": ((16, 24, 24), 1e6, False, 2.5, 1000, 0.5, 6, 0.75),
    "large": ((8,), 1e4, True, 40, 4096, 1, 32, 300.0),
}


def make(name):
    """The axes, and frequencies, axis and magnitude by a formula of their own."""
    sections, base, adjacent, factor, length, slow, fast, magnitude = CASES[name]
    axes = min_fa3_op.RotaryAxes.from_sections(sections, base, adjacent=adjacent)
    axes = axes.stretched(factor, length, slow=slow, fast=fast, magnitude=magnitude)
    freq, pairs = [], sum(sections)
    for i in range(pairs):
        f = base ** (-i / pairs)
        share = 0.0 if math.isinf(slow) else min(1.0, max(0.0, (length * f / (2 * math.pi) - slow) / (fast - slow)))
        freq.append(share * f + (1 - share) * f / factor)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return axes, freq, axis, 0.1 * math.log(factor) + 1 if magnitude is None else magnitude


def reference(x, positions, name, sign=1):
    """x [..., heads, 128], positions [axes, ...] -> [tokens, heads, 128] in 64 bits."""
    _, freq, axis, magnitude = make(name)
    adjacent = CASES[name][2]
    ref = turn(x.detach().cpu().reshape(-1, *x.shape[-2:]), positions.cpu().reshape(positions.size(0), -1), freq, axis, adjacent, sign)
    ref[..., :2 * len(freq)] *= magnitude
    return ref


def check(ours, x, positions, name, sign=1):
    _, freq, _, magnitude = make(name)
    x, ref = x.detach().double().cpu().reshape(-1, *x.shape[-2:]), reference(x, positions, name, sign)
    ours = ours.detach().double().cpu().reshape(ref.shape)
    slack = ref.abs() * BF16_HALF_STEP * (1 + 2**-10) + 2**-20 * magnitude * x.abs().max().item()
    off = (ours - ref).abs()
    assert (off <= slack).all(), f"off by {(off / slack).max().item():.2f} of the bound"
    assert torch.equal(ours[..., 2 * len(freq):], x[..., 2 * len(freq):]), "dimensions behind the pairs changed"


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("batch,seq,qh,kvh", [(1, 1, 1, 1), (2, 37, 8, 2), (1, 2000, 5, 1)])
def test_turned(name, batch, seq, qh, kvh):
    gen = torch.Generator().manual_seed(seq)
    axes = make(name)[0]
    q, k = randn(gen, batch, seq, qh, 128).cuda(), randn(gen, batch, seq, kvh, 128).cuda()
    positions = torch.randint(0, 10**6, (axes.axes, batch, seq), generator=gen).cuda()
    for inverse in (False, True):
        q_out, k_out = min_fa3_op.rotary(q, k, positions, axes, inverse=inverse)
        check(q_out, q, positions, name, -1 if inverse else 1)
        check(k_out, k, positions, name, -1 if inverse else 1)


@pytest.mark.parametrize("name", ["long", "axes", "large"])
def test_gradients(name):
    """Against the formula, and against differences: the loss is linear in q, so (loss(q + u) - loss(q)) is <dq, u> exactly, up to
    the rounding of dq, half a step a value."""
    gen = torch.Generator().manual_seed(5)
    axes = make(name)[0]
    q, k = randn(gen, 2, 19, 4, 128).cuda().requires_grad_(), randn(gen, 2, 19, 2, 128).cuda().requires_grad_()
    positions = torch.randint(0, 100000, (axes.axes, 2, 19), generator=gen).cuda()
    gq, gk = randn(gen, 2, 19, 4, 128).cuda(), randn(gen, 2, 19, 2, 128).cuda()
    q_out, k_out = autograd.rotary(q, k, positions, axes)
    check(q_out, q, positions, name)
    dq, dk = torch.autograd.grad((q_out, k_out), (q, k), (gq, gk), create_graph=False)
    check(dq, gq, positions, name, -1)
    check(dk, gk, positions, name, -1)
    flat = gq.cpu().reshape(-1, 4, 128).double()
    x, u = q.detach().cpu().reshape(-1, 4, 128).double(), torch.randn(38, 4, 128, generator=gen, dtype=torch.float64)
    there = reference(x + u, positions, name) - reference(x, positions, name)
    slope = (dq.double().cpu().reshape(-1, 4, 128) * u).sum().item()
    off = (dq.double().cpu().reshape(-1, 4, 128) * u).abs().sum().item() * BF16_HALF_STEP
    assert abs((there * flat).sum().item() - slope) <= off * (1 + 2**-6)


def test_gradient_of_the_gradient():
    gen = torch.Generator().manual_seed(7)
    axes = make("long")[0]
    q, g = randn(gen, 10, 2, 128).cuda().requires_grad_(), randn(gen, 10, 2, 128).cuda().requires_grad_()
    positions = torch.randint(0, 1000, (1, 10), generator=gen).cuda()
    dq, = torch.autograd.grad(autograd.rotary(q, None, positions, axes)[0], q, g, create_graph=True)
    u = randn(gen, 10, 2, 128).cuda()
    dg, = torch.autograd.grad(dq, g, u)
    check(dg, u, positions, "long")


def test_captured_backward_while_an_eager_graph_lives():
    gen = torch.Generator().manual_seed(8)
    axes = make("axes")[0]
    leaf = randn(gen, 3, 65, 4, 128).cuda().requires_grad_()
    positions = torch.randint(0, 1000, (3, 3, 65), generator=gen).cuda()
    grad = randn(gen, 3, 65, 4, 128).cuda()
    eager, _ = autograd.rotary(leaf, None, positions, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        mine = leaf.detach().requires_grad_()
        out, _ = autograd.rotary(mine, None, positions, axes)
        d, = torch.autograd.grad(out, mine, grad)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        with torch.no_grad():
            leaf.copy_(randn(gen, 3, 65, 4, 128))
            grad.copy_(randn(gen, 3, 65, 4, 128))
        graph.replay()
        torch.cuda.synchronize()
        check(out, leaf, positions, "axes")
        check(d, grad, positions, "axes", -1)
    assert eager.shape == leaf.shape


def test_traced_step():
    gen = torch.Generator().manual_seed(9)
    axes = make("axes")[0]
    q, k = randn(gen, 2, 33, 4, 128).cuda().requires_grad_(), randn(gen, 2, 33, 2, 128).cuda().requires_grad_()
    positions = torch.randint(0, 9000, (3, 2, 33), generator=gen).cuda()

    def step(a, b):
        return autograd.rotary(a * 2, b, positions, axes)
    want, ours = step(q, k), torch.compile(step, backend="aot_eager", fullgraph=True)(q, k)
    assert all(torch.equal(a, b) for a, b in zip(ours, want))
    grads = [torch.autograd.grad(out, (q, k), [torch.ones_like(t) for t in out]) for out in (ours, want)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("count", [1, 50])
def test_written_into_a_cache_in_16_bits(name, count):
    gen = torch.Generator().manual_seed(count)
    axes = make(name)[0]
    cache, lens = Cache(3, 2, 200, 2, 16), [5, 100]
    q, k, v = randn(gen, 2, count, 4, 128).cuda(), randn(gen, 2, count, 2, 128).cuda(), randn(gen, 2, count, 2, 128).cuda()
    positions = torch.randint(0, 10**6, (axes.axes, 2, count), generator=gen).cuda()
    out = min_fa3_op.append_cache(k, v, cache.k, cache.v, torch.tensor(lens, dtype=torch.int32).cuda(), block_table=cache.table, q=q,
                                  positions=positions, axes=axes)
    min_fa3_op.check_last_status("append_cache")
    check(out, q, positions, name)
    check(torch.stack([cache.rows("k", b, n + count)[n:] for b, n in enumerate(lens)]), k, positions, name)
    for b, n in enumerate(lens):
        assert torch.equal(cache.rows("v", b, n + count)[n:], v[b].double().cpu())
