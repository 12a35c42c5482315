"""Rotary positions on the GPU against the formula in 64 bits: axes, layouts, strides, far positions, gradients, streams, graphs."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import assert_turned, randn, turn
from min_fa3_demo_b200 import autograd

pytestmark = pytest.mark.gpu

LAYOUTS = {
    "text": ((64,), 1e6, False, False),
    "half": ((32,), 1e4, False, True),
    "eight": ((8,), 1e4, False, False),
    "mixed": ((16, 24, 24), 1e6, False, False),
    "image": ((32, 32), 1e4, True, True),
    "video": ((22, 21, 21), 1e4, True, False),
    "odd": ((1, 5, 0, 34), 5e5, True, True),
}


def frequencies(layout):
    sections, base, restart, adjacent = LAYOUTS[layout]
    freq, axis = [], []
    for a, n in enumerate(sections):
        for j in range(n):
            freq.append(base ** (-(j / n if restart else len(freq) / sum(sections))))
            axis.append(a)
    return freq, axis, adjacent


def make(layout):
    sections, base, restart, adjacent = LAYOUTS[layout]
    return min_fa3_op.RotaryAxes.from_sections(sections, base, restart=restart, adjacent=adjacent)


def check(ours, x, positions, layout, sign=1):
    freq, axis, adjacent = frequencies(layout)
    flat = x.detach().cpu().reshape(-1, *x.shape[-2:])
    ref = turn(flat, positions.cpu().reshape(positions.size(0), -1), freq, axis, adjacent, sign)
    assert_turned(ours.detach().reshape(flat.shape), flat, ref, len(freq))


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("batch,seq,qh,kvh", [(1, 1, 1, 1), (2, 37, 8, 2), (3, 700, 5, 1)])
def test_layouts_and_sizes(layout, batch, seq, qh, kvh):
    gen = torch.Generator().manual_seed(seq)
    axes = make(layout)
    q, k = randn(gen, batch, seq, qh, 128).cuda(), randn(gen, batch, seq, kvh, 128).cuda()
    positions = torch.randint(0, 5000, (axes.axes, batch, seq), generator=gen).cuda()
    for inverse in (False, True):
        q_out, k_out = min_fa3_op.rotary(q, k, positions, axes, inverse=inverse)
        check(q_out, q, positions, layout, -1 if inverse else 1)
        check(k_out, k, positions, layout, -1 if inverse else 1)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_far_and_negative_positions(dtype):
    # 32-bit angles would be off by whole radians here.  64-bit ones (the reference) are off by 2^31 * 2^-53.
    gen = torch.Generator().manual_seed(1)
    q = randn(gen, 6, 3, 128).cuda()
    positions = torch.tensor([[0, -1, 2**31 - 1, -2**31, 123456789, 1_000_003]], dtype=dtype).cuda()
    check(min_fa3_op.rotary(q, None, positions, make("text"))[0], q, positions, "text")


def test_frequencies_of_more_than_a_turn_and_none():
    gen = torch.Generator().manual_seed(2)
    freq = [0.0, -0.5, 7.25, 1e-9, 3.0, 1.0, 2.0, 100.0]
    axes = min_fa3_op.RotaryAxes(freq, adjacent=True)
    q = randn(gen, 200, 2, 128).cuda()
    positions = torch.arange(200).cuda()[None]
    out, none = min_fa3_op.rotary(q, None, positions, axes)
    assert none is None
    assert_turned(out, q.cpu(), turn(q.cpu(), positions.cpu(), freq, [0] * 8, True), 8)
    assert torch.equal(out[..., :2], q[..., :2])          # frequency 0


@pytest.mark.parametrize("view", ["fused", "heads first", "one in three", "expanded"])
def test_strided_inputs(view):
    gen = torch.Generator().manual_seed(3)
    axes = make("mixed")
    if view == "fused":
        both = randn(gen, 2, 33, 6, 128).cuda()
        q, k = both[:, :, :4], both[:, :, 4:]
    elif view == "heads first":
        q, k = (randn(gen, 2, h, 33, 128).cuda().transpose(1, 2) for h in (4, 2))
    elif view == "one in three":
        q, k = randn(gen, 2, 99, 4, 128).cuda()[:, ::3], randn(gen, 2, 33, 2, 384).cuda()[..., 128:256]
    else:
        q, k = randn(gen, 1, 33, 4, 128).cuda().expand(2, -1, -1, -1), randn(gen, 2, 33, 1, 128).cuda().expand(-1, -1, 3, -1)
    positions = torch.randint(0, 9000, (3, 1, 33), generator=gen).cuda().expand(-1, 2, -1)   # one row for the whole batch
    q_out, k_out = min_fa3_op.rotary(q, k, positions, axes)
    assert q_out.is_contiguous() and k_out.is_contiguous()
    check(q_out, q, positions, "mixed")
    check(k_out, k, positions, "mixed")


def test_nothing_spreads_from_pair_to_pair():
    gen = torch.Generator().manual_seed(4)
    axes = min_fa3_op.RotaryAxes.from_sections((32,))
    clean = randn(gen, 40, 3, 128)
    q = clean.clone()
    q[7, 1, 5], q[9, 2, 100], q[11, 0, 127] = float("nan"), float("inf"), float("-inf")
    positions = torch.arange(40).cuda()[None]
    out = min_fa3_op.rotary(q.cuda(), None, positions, axes)[0].cpu()
    good = min_fa3_op.rotary(clean.cuda(), None, positions, axes)[0].cpu()
    touched = torch.zeros(40, 3, 128, dtype=torch.bool)
    touched[7, 1, 5] = touched[7, 1, 37] = touched[9, 2, 100] = touched[11, 0, 127] = True
    assert torch.equal(out[~touched], good[~touched])
    assert out[7, 1, 5].isnan() and out[7, 1, 37].isnan()
    assert out[9, 2, 100] == float("inf") and out[11, 0, 127] == float("-inf")       # not turned: copied


def test_empty_inputs():
    axes = make("image")
    q, k = min_fa3_op.rotary(torch.empty(2, 0, 4, 128, dtype=torch.bfloat16, device="cuda"), None,
                             torch.empty(2, 2, 0, dtype=torch.int64, device="cuda"), axes)
    assert q.shape == (2, 0, 4, 128) and k is None


@pytest.mark.parametrize("layout", ["mixed", "image", "half"])
def test_gradients(layout):
    """Against the formula, and against differences: the loss is linear in q, so (loss(q + u) - loss(q)) is <dq, u> exactly, up to
    the rounding of dq, half a step a value."""
    gen = torch.Generator().manual_seed(5)
    axes = make(layout)
    freq, axis, adjacent = frequencies(layout)
    q, k = randn(gen, 2, 19, 4, 128).cuda().requires_grad_(), randn(gen, 2, 19, 2, 128).cuda().requires_grad_()
    positions = torch.randint(0, 100000, (axes.axes, 2, 19), generator=gen).cuda()
    gq, gk = randn(gen, 2, 19, 4, 128).cuda(), randn(gen, 2, 19, 2, 128).cuda()
    q_out, k_out = autograd.rotary(q, k, positions, axes)
    dq, dk = torch.autograd.grad((q_out, k_out), (q, k), (gq, gk))
    check(dq, gq, positions, layout, -1)
    check(dk, gk, positions, layout, -1)
    flat, where = gq.cpu().reshape(-1, 4, 128).double(), positions.cpu().reshape(axes.axes, -1)
    x, u = q.detach().cpu().reshape(-1, 4, 128).double(), torch.randn(38, 4, 128, generator=gen, dtype=torch.float64)

    def loss(z):
        return (turn(z, where, freq, axis, adjacent) * flat).sum().item()
    slope = (dq.double().cpu().reshape(-1, 4, 128) * u).sum().item()
    off = (dq.double().cpu().reshape(-1, 4, 128) * u).abs().sum().item() * torch.finfo(torch.bfloat16).eps / 2
    assert abs(loss(x + u) - loss(x) - slope) <= off * (1 + 2**-6)


def test_gradients_of_one_output_only_and_of_layouts():
    gen = torch.Generator().manual_seed(6)
    axes = make("text")
    q, k = randn(gen, 50, 4, 128).cuda().requires_grad_(), randn(gen, 50, 2, 128).cuda().requires_grad_()
    positions = torch.arange(50).cuda()[None]
    q_out, k_out = autograd.rotary(q, k, positions, axes)
    k_out.float().sum().backward()                        # an expanded gradient, and none for q
    assert q.grad is None
    check(k.grad, torch.ones_like(k), positions, "text", -1)
    k.grad = None
    q_out, _ = autograd.rotary(q, None, positions, axes)
    g = randn(gen, 50, 128, 4).cuda().transpose(1, 2)     # a gradient whose heads' values are not adjacent
    dq, = torch.autograd.grad(q_out, q, g)
    check(dq, g, positions, "text", -1)
    # A broadcast input: the gradient of a head shared by four is the sum over them.
    one = randn(gen, 50, 1, 128).cuda().requires_grad_()
    out, _ = autograd.rotary(one.expand(-1, 4, -1), None, positions, axes)
    d, = torch.autograd.grad(out, one, torch.ones_like(out))
    each = min_fa3_op.rotary(torch.ones_like(out), None, positions, axes, inverse=True)[0]
    assert torch.equal(d, each.sum(1, keepdim=True))


def test_gradient_of_the_gradient():
    gen = torch.Generator().manual_seed(7)
    axes = make("mixed")
    q = randn(gen, 10, 2, 128).cuda().requires_grad_()
    positions = torch.randint(0, 1000, (3, 10), generator=gen).cuda()
    g = randn(gen, 10, 2, 128).cuda().requires_grad_()
    dq, = torch.autograd.grad(autograd.rotary(q, None, positions, axes)[0], q, g, create_graph=True)
    u = randn(gen, 10, 2, 128).cuda()
    dg, = torch.autograd.grad(dq, g, u)
    check(dg, u, positions, "mixed")


def test_stream_graph_and_repeated_calls():
    gen = torch.Generator().manual_seed(8)
    axes = make("mixed")
    q, k = randn(gen, 3, 65, 8, 128).cuda(), randn(gen, 3, 65, 2, 128).cuda()
    positions = torch.randint(0, 1000, (3, 3, 65), generator=gen).cuda()
    want = min_fa3_op.rotary(q, k, positions, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        there = min_fa3_op.rotary(q, k, positions, axes)
        leaf = q.clone().requires_grad_()
        with torch.cuda.graph(graph, stream=side):
            captured = min_fa3_op.rotary(q, k, positions, axes)
            out, _ = autograd.rotary(leaf, None, positions, axes)
            grad, = torch.autograd.grad(out, leaf, q)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, want))
    for _ in range(2):
        q.copy_(randn(gen, 3, 65, 8, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, min_fa3_op.rotary(q, k, positions, axes)))
        assert torch.equal(grad, min_fa3_op.rotary(q, None, positions, axes, inverse=True)[0])
