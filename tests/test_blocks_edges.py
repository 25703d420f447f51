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


@pytest.mark.gpu
def test_out_is_seen_as_written():
    """A tensor that autograd saved may not be overwritten behind its back."""
    a, b = t5.quantize_blocks(make(1, 40, 64)), t5.quantize_blocks(make(2, 64, 64))

    def product(out):
        t5.block_scaled_mm(a, b, dtype=torch.float32, out=out)

    def values(out):
        t5.dequantize_blocks(a, out=out)

    for write in (product, values):
        buffer = make(3, 40, 64)
        w = torch.ones(40, 64, device="cuda", requires_grad=True)
        z = w * buffer
        version = buffer._version
        write(buffer)
        assert buffer._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        # a part of a larger tensor counts for the whole
        big = make(4, 50, 80)
        z = w * big[5:45, 8:72]
        write(big[5:45, 8:72])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        # a refused call writes nothing and counts nothing
        version = big._version
        with pytest.raises(ValueError):
            write(big[5:45, 8:71])
        assert big._version == version
        with torch.inference_mode():
            held = torch.zeros(40, 64, device="cuda")
            write(held)
            assert bool(held.any())
            held.zero_()
        with pytest.raises(RuntimeError, match="[Ii]nference tensor"):
            write(held)
        assert not bool(held.any())
