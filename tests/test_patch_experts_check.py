"""Experts modules whose own forward is not the kernels' layer are refused by the 4-bit patches, as patch_dense refuses them."""
import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import patch  # noqa: E402
from test_patch import D, KINDS, _init, make_block  # noqa: E402


def clamped(block):
    """SiLU by its name, with gates and ups that are cut off."""
    class Experts(type(block.experts)):
        def forward(self, hidden_states, top_k_index, top_k_weights):
            y = torch.zeros_like(hidden_states)
            for j in range(top_k_index.shape[1]):
                gu = torch.einsum("td,tfd->tf", hidden_states, self.gate_up_proj[top_k_index[:, j]])
                g, u = gu.chunk(2, -1)
                h = self.act_fn(g.clamp(max=7.0)) * u.clamp(-7.0, 7.0)
                y += top_k_weights[:, j:j + 1] * torch.einsum("tf,tdf->td", h, self.down_proj[top_k_index[:, j]])
            return y
    block.experts.__class__ = Experts
    return block


def test_clamped_experts():
    block = clamped(make_block("mixtral", "cpu"))
    for call in (patch.patch_block, lambda b: patch.patch_experts(b.experts)):
        with pytest.raises(ValueError, match="clamp"):
            call(block)
    assert not hasattr(block, "_moelab_state") and not hasattr(block.experts, "_moelab_state")


@pytest.mark.parametrize("act,kernel", [("silu", 0), ("gelu_pytorch_tanh", 1), ("gelu", 1)])
def test_plain_layers_are_taken(act, kernel):
    """The exact GELU is as near to the kernels' as 4-bit weights let anyone see."""
    from transformers.models.mixtral.configuration_mixtral import MixtralConfig
    from transformers.models.mixtral.modeling_mixtral import MixtralSparseMoeBlock
    cfg = MixtralConfig(hidden_size=D, intermediate_size=320, num_local_experts=4, num_experts_per_tok=2, hidden_act=act)
    assert patch._glu_of(_init(MixtralSparseMoeBlock(cfg), "cpu").experts) == kernel


@pytest.mark.parametrize("kind", [k for k in KINDS if k != "gpt-oss"])
def test_families(kind):
    assert patch._glu_of(make_block(kind, "cpu").experts) == 0


def test_gptoss_form():
    """Another clamp, or gate and up one behind the other, under gpt-oss's names."""
    assert patch.block_state(make_block("gpt-oss", "cpu"))["act"] == 2
    block = make_block("gpt-oss", "cpu")

    class Experts(type(block.experts)):
        def forward(self, *args, **kw):
            order = torch.cat([torch.arange(0, 64, 2), torch.arange(1, 64, 2)]).argsort()
            self.gate_up_proj = torch.nn.Parameter(self.gate_up_proj[..., order], requires_grad=False)
            self.gate_up_proj_bias = torch.nn.Parameter(self.gate_up_proj_bias[..., order], requires_grad=False)
            return super().forward(*args, **kw)
    block.experts.__class__ = Experts
    with pytest.raises(ValueError, match="interleaved"):
        patch.block_state(block)
    block = make_block("gpt-oss", "cpu")
    block.experts.limit = 5.0
    with pytest.raises(ValueError, match="interleaved"):
        patch.block_state(block)
