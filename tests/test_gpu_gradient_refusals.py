"""Incoming gradients that raw pointers cannot stand for are refused: tangents, batches of gradients, subclasses."""
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from peco_amd import rotary, window
from peco_amd.rotary import RotaryAxes, rotary_axes
from peco_amd.window import window_attention

AXES = RotaryAxes((16, 24, 24))


class Tagged(torch.Tensor):
    pass


def _calls(device):
    g = torch.Generator().manual_seed(1)
    leaves = [torch.randn(1, 2, 50, 64, generator=g).to(device, torch.bfloat16).requires_grad_() for _ in range(3)]
    positions = RotaryAxes.grid(2, 5, 5, device=device)
    return {"window": (leaves, lambda: window_attention(*leaves, (10, 0), 2)),
            "rotary": (leaves[:1], lambda: rotary_axes(leaves[0], positions, AXES))}


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["window", "rotary"])
def test_gradients_refused(name, announce):
    """A tangent of the incoming gradient would be lost without a word: the gradients are linear in it."""
    announce()
    leaves, call = _calls("cuda:0")[name]
    out = call()
    grad = torch.randn_like(out)
    want = torch.autograd.grad(out, leaves, grad, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="ordinary"):
            torch.autograd.grad(out, leaves, forward_ad.make_dual(grad, torch.randn_like(grad)), retain_graph=True)
        again = torch.autograd.grad(out, leaves, grad, retain_graph=True)  # (no tangent: taken, inside a level too)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    with pytest.raises(RuntimeError, match="ordinary"):
        torch.autograd.grad(out, leaves, torch.stack([grad, grad]), is_grads_batched=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="ordinary"):
        torch.autograd.grad(out, leaves, grad.as_subclass(Tagged), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, grad), want))


@pytest.mark.parametrize("kind", ["tangent", "subclass"])
def test_backward_functions_refuse_before_a_launch(kind):
    """No launch is reached: this runs without a GPU."""
    q, grad = torch.zeros(1, 2, 5, 64).bfloat16(), torch.zeros(1, 2, 5, 64).bfloat16()
    saved = SimpleNamespace(saved_tensors=(q, q, q, None, q, q, q, q), mask=(1, 0, 0, 0.125))
    turned = SimpleNamespace(saved_tensors=(torch.zeros(3, 5, dtype=torch.int32),), axes=AXES)
    with forward_ad.dual_level():
        grad = forward_ad.make_dual(grad, grad + 1) if kind == "tangent" else grad.as_subclass(Tagged)
        with pytest.raises(RuntimeError, match="ordinary"):
            window._WindowAttention.backward(saved, grad)
        with pytest.raises(RuntimeError, match="ordinary"):
            rotary._RotaryAxes.backward(turned, grad)
