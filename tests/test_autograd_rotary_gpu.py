"""``autograd.rotary`` on the GPU: inputs and gradients that the kernels cannot take as they are."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import randn
from min_fa3_demo_b200 import autograd

pytestmark = pytest.mark.gpu

AXES = min_fa3_op.RotaryAxes.from_sections((16, 24, 24))


def odd_address(t):
    """The same values, contiguous, 2 bytes behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    there = flat[1:1 + t.numel()].view(t.shape)
    there.copy_(t)
    assert there.is_contiguous() and there.data_ptr() % 16 == 2
    return there


def test_addresses_that_are_not_aligned_and_zero_tensors():
    gen = torch.Generator().manual_seed(1)
    q, k, g = (randn(gen, 2, 33, h, 128).cuda() for h in (4, 2, 4))
    positions = torch.randint(0, 9000, (3, 2, 33), generator=gen).cuda()
    want_q, want_k = min_fa3_op.rotary(q, k, positions, AXES)
    leaf = odd_address(q).requires_grad_()
    out, out_k = autograd.rotary(leaf, odd_address(k), positions, AXES)
    assert torch.equal(out, want_q) and torch.equal(out_k, want_k)
    back = min_fa3_op.rotary(g, None, positions, AXES, inverse=True)[0]
    assert torch.equal(torch.autograd.grad(out, leaf, odd_address(g), retain_graph=True)[0], back)
    negated = torch.autograd.grad(out, leaf, torch._neg_view(odd_address(g)), retain_graph=True)[0]
    assert torch.equal(negated, -back)
    zero = torch._efficientzerotensor(out.shape, dtype=out.dtype, device=out.device)
    grad, = torch.autograd.grad(out, leaf, zero)
    assert grad.shape == q.shape and not grad.any()


def test_fake_tensors_and_a_traced_step():
    """As ``attention``: a compiled step has the operator in its graph, and gives the bits of the ordinary one."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = (torch.empty(2, 33, h, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True) for h in (4, 2))
        out, out_k = autograd.rotary(q, k, torch.empty(3, 2, 33, dtype=torch.int64, device="cuda"), AXES)
        grads = torch.autograd.grad((out, out_k), (q, k), (out, out_k))
        assert [t.shape for t in (out, out_k, *grads)] == [q.shape, k.shape] * 2
    gen = torch.Generator().manual_seed(2)
    q, k, v = (randn(gen, 2, 33, h, 128).cuda().requires_grad_() for h in (4, 2, 2))
    positions = torch.randint(0, 9000, (3, 2, 33), generator=gen).cuda()

    # Three tensors: a compiled autograd.Function whose arguments are one tensor twice loses a gradient, whatever it computes.
    def step(a, b, c):
        out, out_k = autograd.rotary(a * 2, b, positions, AXES)
        return autograd.attention(out, out_k, c, True, deterministic=True)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    want, ours = step(q, k, v), compiled(q, k, v)
    assert torch.equal(ours, want)
    for a, b in zip(torch.autograd.grad(ours, (q, k, v), torch.ones_like(ours)), torch.autograd.grad(want, (q, k, v), torch.ones_like(want))):
        assert torch.equal(a, b)


def test_profilers_see_the_operator():
    q = torch.zeros(5, 4, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    positions = torch.zeros(3, 5, dtype=torch.int64, device="cuda")
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        autograd.rotary(q, None, positions, AXES)[0].sum().backward()
    assert "b200attn::rotary" in {e.key for e in prof.key_averages()}
