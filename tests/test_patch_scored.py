"""Group-limited and sigmoid gates of patched blocks on router.route_scored: which gates it takes, and the patched block against the
stock one on the same weights."""
import pytest
import torch

from moelab_amd import patch
from test_patch import D, _init, make_block


def sigmoid_block(device, bias=0.0, **kw):
    """DeepSeek-V3's block, its choice bias random around `bias`."""
    from transformers.models.deepseek_v3.configuration_deepseek_v3 import DeepseekV3Config
    from transformers.models.deepseek_v3.modeling_deepseek_v3 import DeepseekV3MoE
    cfg = DeepseekV3Config(**(dict(hidden_size=D, moe_intermediate_size=256, n_routed_experts=16, num_experts_per_tok=4, n_group=4,
                                   topk_group=2, n_shared_experts=1, routed_scaling_factor=2.5, norm_topk_prob=True) | kw))
    block = _init(DeepseekV3MoE(cfg), device)
    with torch.no_grad():
        b = block.gate.e_score_correction_bias
        b.copy_(bias + 0.2 * torch.rand(b.shape, generator=torch.Generator().manual_seed(5)))
    return block


def settings(block):
    return patch._scored_settings(block.gate, block.gate.top_k)


def test_which_gates():
    assert settings(make_block("deepseek-group", "cpu")) == dict(score="softmax", group_score="max", norm=False, groups=2, top_groups=1,
                                                                scale=2.5)
    want = dict(score="sigmoid", group_score="top2", norm=True, groups=4, top_groups=2, scale=2.5)
    assert settings(sigmoid_block("cpu")) == want
    assert settings(sigmoid_block("cpu", norm_topk_prob=False)) == want | dict(norm=False)
    assert settings(sigmoid_block("cpu", n_group=1, topk_group=1)) == want | dict(groups=1, top_groups=1)
    # masked groups at 0 win over kept experts below 0: only where no group is masked
    assert settings(sigmoid_block("cpu", bias=-0.3)) is None
    assert settings(sigmoid_block("cpu", bias=-0.3, n_group=1, topk_group=1)) is not None


def test_a_gate_that_does_something_else_stays_stock():
    block = make_block("deepseek-group", "cpu")

    class Other(type(block.gate)):
        def forward(self, x):
            out = super().forward(x)
            return out[0], out[1] * 1.01, out[2]
    block.gate.__class__ = Other
    assert settings(block) is None

    class Broken(type(block.gate)):
        def forward(self, x, more):
            raise AssertionError
    block.gate.__class__ = Broken
    assert settings(block) is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["groups", "sigmoid", "sigmoid, one group", "negative bias"])
@pytest.mark.parametrize("T", [1, 24])
def test_patched_block_matches_stock(kind, T):
    from helpers import assert_close
    block = {"groups": lambda: make_block("deepseek-group", "cuda"), "sigmoid": lambda: sigmoid_block("cuda"),
             "sigmoid, one group": lambda: sigmoid_block("cuda", n_group=1, topk_group=1),
             "negative bias": lambda: sigmoid_block("cuda", bias=-0.3)}[kind]()
    x = torch.randn(1, T, D, generator=torch.Generator().manual_seed(T)).to("cuda", torch.bfloat16)
    patch.patch_block(block)
    cfg = block._moelab_cfg
    assert cfg["stock_gate"] and (cfg["scored"] is None) == (kind == "negative bias")
    calls = []
    stock = type(block.gate).forward

    class Counted(type(block.gate)):
        def forward(self, x):
            calls.append(1)
            return stock(self, x)
    block.gate.__class__ = Counted
    block.float()   # the stock modules in fp32, so the dequantised weights land exactly
    patch.load_dequantised(block)
    with torch.no_grad():
        flat = x.reshape(-1, D).float()
        out = block.gate(flat)
        ref = block.experts(flat, out[2].long(), out[1].float()) + block.shared_experts(flat)
        for gate, own in ((torch.bfloat16, cfg["scored"] is not None), (torch.float32, False)):
            block.gate.to(gate)
            calls.clear()
            y = block(x) if gate == torch.bfloat16 else block(x.float())
            assert len(calls) == (0 if own else 1), (gate, calls)
            assert_close(y.reshape(-1, D), ref.cpu().numpy(), what=("patch", kind, T, gate))
        seen = []   # a gate with a hook runs
        block.gate.to(torch.bfloat16).register_forward_hook(lambda *a: seen.append(1))
        block(x)
        assert seen


@pytest.mark.gpu
def test_the_gates_bias_is_read_when_it_is_used():
    block = sigmoid_block("cuda")
    patch.patch_block(block)
    x = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    with torch.no_grad():
        first = block(x)
        block.gate.e_score_correction_bias.copy_(block.gate.e_score_correction_bias.flip(0) * 5)
        assert not torch.equal(first, block(x))


@pytest.mark.gpu
def test_a_bias_that_becomes_negative_brings_the_gate_back():
    """Also in a graph that is captured after the change, where the bias cannot be looked at."""
    block = sigmoid_block("cuda")
    patch.patch_block(block)
    x = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    calls = []
    stock = type(block.gate).forward

    class Counted(type(block.gate)):
        def forward(self, x):
            calls.append(1)
            return stock(self, x)
    block.gate.__class__ = Counted
    bias = block.gate.e_score_correction_bias
    with torch.no_grad():
        for shift, own in ((0.0, True), (-1.0, False), (1.0, True), (0.5, True)):
            bias += shift
            calls.clear()
            block(x)
            assert len(calls) == (0 if own else 1), shift
        calls.clear()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(x)
        assert not calls
        eager = block(x)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


@pytest.mark.gpu
def test_hidden_states_that_require_grad():
    """A patched block has no backward pass; with gradients enabled it still runs."""
    block = sigmoid_block("cuda")
    patch.patch_block(block)
    x = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    with torch.no_grad():
        want = block(x)
    assert torch.equal(block(x.requires_grad_()), want)
