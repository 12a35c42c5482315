"""``autograd.rotary`` without a GPU: what it makes of tensors that the kernels cannot take as they are."""
from __future__ import annotations

import contextlib

import pytest
import torch

from min_fa3_demo_b200 import autograd as ag

BF16 = torch.bfloat16


def odd_address(*shape):
    """Contiguous values that begin 2 bytes behind a 16-byte boundary."""
    flat = torch.randn(torch.Size(shape).numel() + 8).to(BF16)
    start = next(i for i in range(8) if (flat.data_ptr() + 2 * i) % 16 == 2)
    return flat[start:start + torch.Size(shape).numel()].view(shape)


@pytest.mark.parametrize("what", ["odd address", "expanded", "transposed", "odd rows", "negated", "zero"])
@pytest.mark.parametrize("shape", [(5, 2, 128), (3, 5, 2, 128)])
def test_rows_are_brought_in_order(what, shape):
    t = {"odd address": lambda: odd_address(*shape),
         "expanded": lambda: torch.randn(*shape[:-1], 1).to(BF16).expand(shape),
         "transposed": lambda: torch.randn(*shape[:-2], 128, shape[-2]).to(BF16).transpose(-1, -2),
         "odd rows": lambda: torch.randn(*shape[:-1], 132).to(BF16)[..., :128],
         "negated": lambda: torch._neg_view(odd_address(*shape)),
         "zero": lambda: torch._efficientzerotensor(shape, dtype=BF16)}[what]()
    ours = ag._rows_in_order(t)
    assert ours.shape == t.shape and ours.dtype == BF16 and not ours.is_neg() and not ours._is_zerotensor()
    assert ours.stride(-1) == 1 and ours.data_ptr() % 16 == 0 and ours.data_ptr() != 0
    assert all(s % 8 == 0 for s in ours.stride()[:-1])
    assert torch.equal(ours, torch.zeros(shape, dtype=BF16) if what == "zero" else t.clone())


def test_rows_in_order_stay_where_they_are():
    for t in (torch.zeros(3, 5, 2, 128, dtype=BF16), torch.zeros(3, 5, 6, 128, dtype=BF16)[:, :, 1:3]):
        assert ag._rows_in_order(t) is t


def test_cpu_tensors_and_other_shapes_are_refused_with_words():
    axes = ag._op.RotaryAxes([1.0] * 8)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ag.rotary(torch.zeros(3, 2, 128, dtype=BF16), None, torch.zeros(1, 3, dtype=torch.int64), axes)
    for t in (torch.zeros(128, dtype=BF16), torch.zeros(2, 128, dtype=BF16)):
        assert ag._rows_in_order(t) is t                   # the call's own checks say what is wrong


@pytest.mark.parametrize("need_q,need_k", [(True, True), (True, False), (False, True)])
def test_only_gradients_that_are_asked_for_are_turned(monkeypatch, need_q, need_k):
    turned = []

    def rotary(q, k, positions, axes, *, inverse=False):
        turned.append([h.size(-2) for h in (q, k) if h is not None])
        return q * 2, None if k is None else k * 2
    monkeypatch.setattr(ag, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(ag._op, "rotary", rotary)
    q, k = torch.randn(3, 4, 128, requires_grad=need_q), torch.randn(3, 2, 128, requires_grad=need_k)
    axes = ag._op.RotaryAxes([1.0] * 8)
    for create_graph in (False, True):
        del turned[:]
        out, out_k = ag.rotary(q, k, torch.zeros(1, 3, dtype=torch.int64), axes)
        leaves = [t for t, need in ((q, need_q), (k, need_k)) if need]
        grads = torch.autograd.grad(out.sum() + out_k.sum(), leaves, create_graph=create_graph)
        assert turned == [[4, 2], [h for h, need in ((4, need_q), (2, need_k)) if need]]
        assert all(torch.equal(g, torch.full_like(g, 2)) for g in grads)


def test_lookers_on_see_the_operator(monkeypatch):
    """Meta and fake tensors, tracers and dispatch modes see ``b200attn::rotary``, forward and backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    axes = ag._op.RotaryAxes.from_sections((16, 24, 24), 1e6, adjacent=True)
    target = torch.ops.b200attn.rotary.default

    def step(q, k, positions):
        out, out_k = ag.rotary(q, k, positions, axes)
        return (out, out_k, *torch.autograd.grad((out, out_k), (q, k), (out, out_k)))
    for mode in (contextlib.nullcontext(), FakeTensorMode()):
        with mode:
            q, k = (torch.empty(3, 5, h, 128, dtype=BF16, device="meta") for h in (4, 2))
            positions = torch.empty(3, 3, 5, dtype=torch.int64, device="meta")
            for given in ((q.transpose(0, 1).contiguous().transpose(0, 1), k), (q[:1].expand(3, -1, -1, -1), k)):
                a, b = (g.detach().requires_grad_() for g in given)
                for result, like in zip(step(a, b, positions), (q, k, q, k)):
                    assert result.shape == like.shape and result.is_contiguous() and result.dtype == BF16
    with FakeTensorMode():                                 # an engine for "cuda" needs a GPU, so no gradients here
        q = torch.empty(5, 4, 128, dtype=BF16, device="cuda:0")
        assert ag.rotary(q, None, torch.empty(3, 5, dtype=torch.int64, device="cuda:0"), axes)[0].shape == q.shape
    with FakeTensorMode():
        q, k = (torch.empty(3, 5, h, 128, dtype=BF16, device="meta") for h in (4, 2))
        positions = torch.empty(3, 3, 5, dtype=torch.int64, device="meta")
        graph = make_fx(lambda a, b, p: step(a.requires_grad_(), b.requires_grad_(), p))(q, k, positions).graph
        alone = make_fx(lambda a, p: ag.rotary(a, None, p, axes)[0])(q, positions).graph
    calls = [n for n in graph.nodes if n.target is target]
    assert [n.args[-1] for n in calls] == [False, True] and len([n for n in alone.nodes if n.target is target]) == 1
    turn, axis, adjacent, _ = calls[0].args[3:]
    again = ag._op.RotaryAxes._from_plain(turn, axis, adjacent)
    assert bytes(again._c) == bytes(axes._c) and (again.axes, again.pairs) == (3, 64)


def test_the_operator_gives_the_kernels_the_same_axes(monkeypatch):
    seen = []

    def rotary(q, k, positions, axes, *, inverse=False):
        seen.append((bytes(axes._c), inverse, k is None))
        return q * 2, None if k is None else k * 2
    monkeypatch.setattr(ag, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(ag._op, "rotary", rotary)
    q, k = torch.randn(3, 4, 128), torch.randn(3, 2, 128)
    positions = torch.zeros(2, 3, dtype=torch.int64)
    axes = ag._op.RotaryAxes([-1.0, 0.5, 3.0, 2.0**-20, 0.0, 1e5, -0.3, 0.1], [1, 0] * 4)
    for plain in (True, False):
        for other in (k, None):
            out, out_k = ag._turned(q, other, positions, axes, False, plain)
            assert torch.equal(out, q * 2) and (out_k is None if other is None else torch.equal(out_k, k * 2))
    assert seen == [(bytes(axes._c), False, False), (bytes(axes._c), False, True)] * 2
    with pytest.raises(RuntimeError, match="axes must be a RotaryAxes"):
        ag.rotary(q, k, positions, None)
