"""Block-scaled calls: what autograd sees of them, extreme factors, aliases and moved memory, and roundings value by
value in the tensors' own types."""

from __future__ import annotations

import pytest
import torch

import tcgen05_b200 as t5
from test_blocks import make

# ------------------------------------------------------------ autograd


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "w", "both"])
def test_second_derivative_is_refused_whatever_the_incoming_gradient(which):
    """dx depends on w and dw on x even where the incoming gradient is a constant: a loss of them has to refuse its
    backward pass, not to leave the terms out."""
    x, w = make(1, 20, 64), make(2, 30, 64)
    want = torch.autograd.grad(t5.block_scaled_linear(*(p := [t.clone().requires_grad_() for t in (x, w)])).sum(), p)
    x.requires_grad_(which != "w")
    w.requires_grad_(which != "x")
    leaves = [t for t in (x, w) if t.requires_grad]
    for weight in (None, torch.ones(20, 30, device="cuda")):
        y = t5.block_scaled_linear(x, w)
        out = y.sum() if weight is None else y
        got = torch.autograd.grad(out, leaves, weight, create_graph=True)
        for t, g in zip(leaves, got):
            assert g.requires_grad and torch.equal(g, want[0] if t is x else want[1])
            with pytest.raises(RuntimeError, match="differentiable once"):
                (y.square().sum() + g.square().sum()).backward(retain_graph=True)
        # what does not use them is differentiated as ever
        first = torch.autograd.grad(y.square().sum(), leaves)
        assert all(bool(t.isfinite().all()) and not t.requires_grad for t in first)
