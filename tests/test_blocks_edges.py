"""Block-scaled calls: what autograd sees of them, extreme factors, aliases and moved memory, and roundings value by
value in the tensors' own types."""

from __future__ import annotations

import pytest
import torch

import tcgen05_b200 as t5
from test_blocks import make

# ------------------------------------------------------------ what is kept


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [-1, 0, "both"])
@pytest.mark.parametrize("rows", [1, 70, 0])
def test_a_given_multiplier_is_kept_as_it_was(axis, rows):
    """A program that updates its scale in place does not change what was rounded with it before."""
    if rows == 0 and axis != -1:
        pytest.skip("blocks along an empty axis")
    x = make(1, rows, 96)
    scale = torch.full((1,), 8.0, device="cuda")
    got = t5.quantize_blocks(x, axis=axis, multiplier=scale)
    fixed = t5.quantize_blocks(x, axis=axis, multiplier=8.0)
    scale.fill_(0.25)
    for q, f in zip(got if axis == "both" else (got,), fixed if axis == "both" else (fixed,)):
        assert float(q.multiplier) == 8.0 and q.multiplier.shape == (1,)
        assert torch.equal(t5.dequantize_blocks(q), t5.dequantize_blocks(f))
        if rows:
            assert torch.equal(t5.block_scaled_mm(q, q), t5.block_scaled_mm(f, f))
    # any one-element form of it, and a captured call that reads its value at each replay
    for m in (torch.tensor(8.0, device="cuda"), torch.full((1, 1), 8.0, device="cuda"),
              torch.conj(torch.complex(torch.zeros(1, device="cuda"), torch.full((1,), -8.0, device="cuda"))).imag):
        q = t5.quantize_blocks(x, multiplier=m)
        assert float(q.multiplier) == 8.0
        assert torch.equal(q.data, t5.quantize_blocks(x, multiplier=8.0).data)


@pytest.mark.gpu
def test_a_captured_call_keeps_the_multiplier_of_its_replay():
    x = make(1, 33, 200, dtype=torch.bfloat16)
    scale = torch.full((1,), 2.0, device="cuda")
    t5.quantize_blocks(x, multiplier=scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = t5.quantize_blocks(x, multiplier=scale)
    for m in (4.0, 0.5):
        scale.fill_(m)
        graph.replay()
        scale.fill_(77.0)
        assert float(q.multiplier) == m
        assert torch.equal(t5.dequantize_blocks(q), t5.dequantize_blocks(t5.quantize_blocks(x, multiplier=m)))
