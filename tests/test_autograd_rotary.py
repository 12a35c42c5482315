"""``autograd.rotary`` without a GPU: what it makes of tensors that the kernels cannot take as they are."""
from __future__ import annotations

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
    monkeypatch.setattr(ag, "_plain_tensors", lambda tensors: True, raising=False)
    q, k = torch.randn(3, 4, 128, requires_grad=need_q), torch.randn(3, 2, 128, requires_grad=need_k)
    axes = ag._op.RotaryAxes([1.0] * 8)
    for create_graph in (False, True):
        del turned[:]
        out, out_k = ag.rotary(q, k, torch.zeros(1, 3, dtype=torch.int64), axes)
        leaves = [t for t, need in ((q, need_q), (k, need_k)) if need]
        grads = torch.autograd.grad(out.sum() + out_k.sum(), leaves, create_graph=create_graph)
        assert turned == [[4, 2], [h for h, need in ((4, need_q), (2, need_k)) if need]]
        assert all(torch.equal(g, torch.full_like(g, 2)) for g in grads)
