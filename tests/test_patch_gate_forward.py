"""A forward that is put in a gate's place (as wrappers of modules do), before the block is patched or after, is the one that routes."""
import pytest
import torch

from moelab_amd import patch
from test_patch import D, make_block
from test_patch_scored import sigmoid_block


@pytest.mark.gpu
@pytest.mark.parametrize("when", ["before", "after"])
@pytest.mark.parametrize("kind", ["groups", "sigmoid"])
def test_a_wrapped_gate_runs(kind, when):
    block = make_block("deepseek-group", "cuda") if kind == "groups" else sigmoid_block("cuda")
    calls, stock = [], block.gate.forward

    def wrapped(x):
        calls.append(1)
        return stock(x)
    x = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    if when == "before":
        block.gate.forward = wrapped
    patch.patch_block(block)
    block.gate.forward = wrapped
    calls.clear()
    with torch.no_grad():
        y = block(x)
        assert len(calls) == 1
        del block.gate.forward
        assert len(calls) == 1 and block(x).shape == y.shape and len(calls) == 1


@pytest.mark.gpu
def test_a_gate_whose_settings_change_runs():
    block = sigmoid_block("cuda")
    patch.patch_block(block)
    x = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    with torch.no_grad():
        first = block(x)
        gate = block.gate
        scale, gate.routed_scaling_factor = gate.routed_scaling_factor, 25.0
        assert not torch.allclose(first, block(x), rtol=0.1, atol=0.0)
        gate.routed_scaling_factor = scale
        assert torch.equal(first, block(x))
