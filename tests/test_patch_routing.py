"""A sparse MoE block is patched by what its own forward does: the weights that it gives its experts and what it adds to their result.
Blocks that look like a family and compute something else keep their own forward around the patched experts."""
import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import patch  # noqa: E402
from test_patch import D, KINDS, _init, make_block  # noqa: E402
from test_patch_scored import sigmoid_block  # noqa: E402


def sigmoid_gate(block):
    """The block with a gate that takes sigmoid scores, renormalised."""
    class Gate(type(block.gate)):
        def forward(self, x):
            logits = torch.nn.functional.linear(x.reshape(-1, x.shape[-1]), self.weight)
            wts, idx = torch.sigmoid(logits).topk(self.top_k, dim=-1)
            return logits, wts / wts.sum(-1, keepdim=True), idx
    block.gate.__class__ = Gate
    return block


def changed(block, after=lambda self, x, y: y, before=lambda self, x: x):
    """The block with its tokens or its result changed by its own forward."""
    class Block(type(block)):
        def forward(self, x):
            return after(self, x, super().forward(before(self, x)))
    block.__class__ = Block
    return block


def bias_beside(device):
    """Sigmoid scores and a bias that ranks, which the block holds and not its gate."""
    block = make_block("mixtral", device)

    class Block(type(block)):
        def forward(self, x):
            flat = x.reshape(-1, x.shape[-1])
            s = torch.sigmoid(torch.nn.functional.linear(flat, self.gate.weight)).float()
            idx = (s + self.choice_bias).topk(2, dim=-1).indices
            w = s.gather(1, idx)
            return self.experts(flat, idx, w / w.sum(-1, keepdim=True)).reshape(x.shape)
    block.__class__ = Block
    block.register_buffer("choice_bias", torch.tensor([0.3, 0.0, 0.1, 0.2], device=device))
    return block


def shared_beside(device):
    """Shared experts that are added, but under a gate without the DeepSeek gates' scale."""
    block = make_block("mixtral", device)
    shared = torch.nn.Sequential(torch.nn.Linear(D, D, bias=False), torch.nn.SiLU())
    block.shared_experts = _init(shared, device, seed=3)
    return changed(block, after=lambda self, x, y: y + self.shared_experts(x))


OWN = {"sigmoid gate": lambda d: sigmoid_gate(make_block("mixtral", d)), "bias beside": bias_beside, "shared beside": shared_beside,
       "scaled result": lambda d: changed(make_block("olmoe", d), after=lambda self, x, y: 2.5 * y),
       "residual": lambda d: changed(make_block("qwen3", d), after=lambda self, x, y: x + y),
       "scaled tokens": lambda d: changed(make_block("qwen3", d), before=lambda self, x: 0.5 * x),
       "norm behind": lambda d: changed(make_block("deepseek", d), after=lambda self, x, y: y / (1 + y.abs().amax(-1, keepdim=True))),
       "no shared gate": lambda d: changed(make_block("qwen2-shared", d), after=lambda self, x, y: 0.5 * y)}


def settings(block):
    cfg = patch.block_state(block)
    return {n: v for n, v in cfg.items() if n in ("kind", "norm", "scale", "k", "stock_gate", "scored")}


@pytest.mark.parametrize("kind", [k for k in KINDS if k != "gpt-oss"])
def test_families_are_what_they_were(kind):
    got = settings(make_block(kind, "cpu"))
    assert got["kind"] == KINDS[kind] and got["stock_gate"] == (kind == "deepseek-group")
    assert got["norm"] == (kind in ("qwen3", "mixtral")) and got["scale"] == (2.5 if "deepseek" in kind else 1.0)


def test_sigmoid_gates_of_the_deepseek_kind():
    assert settings(sigmoid_block("cpu"))["scored"] is not None
    got = settings(sigmoid_block("cpu", bias=-0.3))
    assert got["kind"] == "deepseek" and got["stock_gate"] and got["scored"] is None
    got = settings(sigmoid_gate(make_block("deepseek", "cpu")))
    assert got["kind"] == "deepseek" and got["stock_gate"] and got["scored"] is None


@pytest.mark.parametrize("kind", list(OWN))
def test_blocks_that_do_something_else_keep_their_forward(kind):
    got = settings(OWN[kind]("cpu"))
    assert got["kind"] == "own" and not got["stock_gate"] and got["scored"] is None, got


def test_renormalised_or_not_by_what_the_gate_does():
    block = make_block("qwen3", "cpu")
    assert settings(block)["norm"]
    block.gate.norm_topk_prob = False
    assert not settings(block)["norm"]

    class Plain(type(block.gate)):   # whatever its setting says
        def forward(self, x):
            p = torch.softmax(torch.nn.functional.linear(x, self.weight), -1)
            return (p, *p.topk(self.top_k, dim=-1))
    block.gate.__class__ = Plain
    block.gate.norm_topk_prob = True
    assert not settings(block)["norm"]


def test_experts_that_are_called_otherwise_are_refused():
    block = make_block("mixtral", "cpu")

    class Block(type(block)):
        def forward(self, x):
            flat = x.reshape(-1, x.shape[-1])
            _, wts, idx = self.gate(flat)
            return self.experts(flat, idx, wts, x).reshape(x.shape)
    block.__class__ = Block
    with pytest.raises(NotImplementedError, match="patch_experts"):
        patch.block_state(block)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(OWN))
@pytest.mark.parametrize("T", [1, 24])
def test_patched_block_matches_its_own(kind, T):
    from helpers import assert_close
    block = OWN[kind]("cuda")
    stock = block.forward
    x = torch.randn(1, T, D, generator=torch.Generator().manual_seed(T)).to("cuda", torch.bfloat16)
    for _ in range(2):   # a second patch as well
        patch.patch_block(block)
    assert block._moelab_cfg["kind"] == "own" and hasattr(block.experts, "_moelab_state")
    with torch.no_grad():
        assert block(x).dtype == torch.bfloat16 and block(x).shape == x.shape
        block.float()   # the stock modules in fp32, so the dequantised weights land exactly
        patch.load_dequantised(block)
        y = block(x.float())
        patch.unpatch_block(block)
        assert block.forward == stock and not any(n.startswith("_moelab") for m in (block, block.experts) for n in m.__dict__)
        ref = block(x.float())
    assert_close(y.reshape(-1, D), ref.reshape(-1, D).cpu().numpy(), what=("own", kind, T))


@pytest.mark.gpu
def test_patched_model_with_such_a_block():
    blocks = torch.nn.ModuleList([make_block("mixtral", "cuda"), OWN["sigmoid gate"]("cuda")])
    assert patch.patch_model(blocks) == 2 and patch.patch_model(blocks) == 0
    x = torch.randn(1, 5, D, generator=torch.Generator().manual_seed(0)).to("cuda", torch.bfloat16)
    with torch.no_grad():
        assert all(torch.isfinite(b(x)).all() for b in blocks)
