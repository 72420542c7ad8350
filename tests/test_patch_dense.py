"""The unquantised module patch (patch.patch_dense, patch_model with fmt="dense") on transformers' sparse MoE blocks built from
small random configs: which modules it takes and refuses, the patched blocks against the stock modules in 64 bits on the same
routing, and gradients through the patched block: those of the expert layer that it calls, router included."""
import copy

import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
import dense_helpers as H  # noqa: E402
from moelab_amd import dense, patch  # noqa: E402
from test_patch import D, make_block  # noqa: E402

KINDS = ["qwen3", "mixtral", "olmoe", "qwen2-shared", "qwen2-shared-odd", "deepseek", "deepseek-group"]
SHARED = {"qwen2-shared": "shared_expert", "qwen2-shared-odd": "shared_expert", "deepseek": "shared_experts",
          "deepseek-group": "shared_experts"}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("universal", [False, True])
def test_patches_experts_and_shared_and_undoes_it(kind, universal):
    block = make_block(kind, "cpu")
    stock = block.experts.forward
    n = patch.patch_model(torch.nn.ModuleList([block]), fmt="dense", universal=universal)
    assert n == (2 if kind in SHARED and not universal else 1)
    assert block.experts.forward != stock and not hasattr(block, "_moelab_state")
    assert patch.patch_model(torch.nn.ModuleList([block]), fmt="dense", universal=universal) == 0
    with pytest.raises(ValueError, match="packs nothing"):
        patch.load_dequantised(block.experts)
    with pytest.raises(RuntimeError, match="GPU"):
        block.experts(torch.zeros(1, D, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int64), torch.ones(1, 2))
    patch.unpatch_experts(block.experts)
    assert block.experts.forward == stock and not hasattr(block.experts, "_moelab_state")


def test_refusals():
    with pytest.raises(ValueError, match="neither"):
        patch.patch_dense(make_block("gpt-oss", "cpu").experts)
    with pytest.raises(ValueError, match="neither"):
        patch.patch_model(torch.nn.ModuleList([make_block("gpt-oss", "cpu")]), fmt="dense")
    with pytest.raises(ValueError, match="neither"):
        patch.patch_dense(torch.nn.Linear(32, 32))
    with pytest.raises(TypeError, match="float32"):
        patch.patch_dense(make_block("qwen3", "cpu").float().experts)
    e = make_block("qwen3", "cpu").experts
    F = e.down_proj.shape[2] - 8
    e.gate_up_proj = torch.nn.Parameter(e.gate_up_proj[:, :2 * F].contiguous())
    e.down_proj = torch.nn.Parameter(e.down_proj[:, :, :F].contiguous())
    with pytest.raises(ValueError, match="intermediate size"):
        patch.patch_dense(e)
    mlp = make_block("deepseek", "cpu").shared_experts
    mlp.up_proj = torch.nn.Linear(mlp.up_proj.in_features, mlp.up_proj.out_features, bias=True, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="neither"):
        patch.patch_dense(mlp)


def _reference(block, kind, flat, idx, wts):
    """The stock modules in 64 bits, and the magnitudes its products sum: (y, mags)."""
    b = copy.deepcopy(block).cpu().double()
    x, idx, wts = flat.detach().cpu().double(), idx.cpu(), wts.detach().cpu().double()
    y = b.experts(x, idx, wts)
    mags = torch.zeros_like(y)
    gu, dn, F = b.experts.gate_up_proj, b.experts.down_proj, b.experts.down_proj.shape[2]
    for t in range(x.shape[0]):
        for j in range(idx.shape[1]):
            e = int(idx[t, j])
            g, u = (gu[e] @ x[t])[:F], (gu[e] @ x[t])[F:]
            mags[t] += wts[t, j] * (dn[e].abs() @ (torch.nn.functional.silu(g) * u).abs())
    if kind in SHARED:
        m = getattr(b, SHARED[kind])
        h = (torch.nn.functional.silu(m.gate_proj(x)) * m.up_proj(x)).abs()
        s, smags = m(x), h @ m.down_proj.weight.abs().t()
        gate = 1.0
        if kind.startswith("qwen2"):
            assert b.shared_expert_gate(x).abs().max() < 4
            gate = torch.sigmoid(b.shared_expert_gate(x))
        y, mags = y + gate * s, mags + gate * smags
    return y.detach(), mags.detach()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", H.TYPES)
@pytest.mark.parametrize("T", [1, 3, 37])
def test_patched_block(kind, dtype, T):
    block = make_block(kind, "cuda").to(dtype)
    x = H.randn(T, D, dtype=dtype)
    with torch.no_grad():
        _, wts, idx = block.gate(x)[:3]
        ref, mags = _reference(block, kind, x, idx, wts)
        patch.patch_model(torch.nn.ModuleList([block]), fmt="dense")
        out = block(x[None])
    y = (out[0] if isinstance(out, tuple) else out).reshape(T, D)
    # Roundings to 16 bits, each off by at most half a step of its share of mags. Experts: h, the slot's row, the experts' sum,
    # the block's. Shared MLP: its gate half, its up half, their product, its row, the sigmoid, the logit's (below 4: up to
    # four half steps of the sigmoid), their product, the block's sum: eleven. Their products and the fp32 sums: one more.
    H.check(y.cpu(), ref, 12 * H.half_step(dtype) * mags + H.half_step(dtype) * ref.abs() + 64 * H.tiny(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["qwen3", "olmoe", "deepseek"])
@pytest.mark.parametrize("checkpoint", [True, False])
def test_gradients_reach_every_parameter(kind, checkpoint):
    """A training step through the patched block: the gradients are those of the expert layer on the same routing, and the
    router gets its own through the routing weights."""
    block = make_block(kind, "cuda").train()
    patch.patch_model(torch.nn.ModuleList([block]), fmt="dense", checkpoint=checkpoint)
    T, e = 29, block.experts
    x = H.randn(T, D, dtype=torch.bfloat16).requires_grad_()
    dy = H.randn(T, D, dtype=torch.bfloat16, seed=1)
    out = block(x[None])
    (out[0] if isinstance(out, tuple) else out).reshape(T, D).backward(dy)
    for n, p in block.named_parameters():
        assert p.grad is not None and p.grad.shape == p.shape and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, n
    assert torch.isfinite(x.grad).all()
    with torch.no_grad():
        _, wts, idx = block.gate(x)[:3]
    leaves = [x.detach().requires_grad_(), wts.detach().requires_grad_(), e.gate_up_proj.detach().requires_grad_(),
              e.down_proj.detach().requires_grad_()]
    dense.experts_mlp(leaves[0], idx, *leaves[1:], checkpoint=checkpoint).backward(dy)
    assert torch.equal(e.gate_up_proj.grad, leaves[2].grad) and torch.equal(e.down_proj.grad, leaves[3].grad)


@pytest.mark.gpu
def test_an_update_in_place_is_seen():
    """The module's own parameters are read in each call."""
    block = make_block("mixtral", "cuda")
    x = H.randn(5, D, dtype=torch.bfloat16)
    idx, wts = torch.tensor([[0, 1]] * 5, device="cuda"), torch.full((5, 2), 0.5, device="cuda")
    patch.patch_dense(block.experts)
    with torch.no_grad():
        a = block.experts(x, idx, wts)
        block.experts.down_proj.mul_(2.0)
        assert torch.equal(block.experts(x, idx, wts), 2 * a)


@pytest.mark.gpu
def test_ids_past_32_bits_are_outside():
    e = make_block("mixtral", "cuda").experts
    x = H.randn(3, D, dtype=torch.bfloat16)
    far = torch.tensor([[0, 2 ** 32 + 1], [2 ** 32, 2 ** 33], [-2 ** 32, 3]], device="cuda")
    near = torch.tensor([[0, -1], [-1, 4], [-1, 3]], device="cuda")
    wts = torch.full((3, 2), 0.5, device="cuda")
    with torch.no_grad():
        y = dense.experts_mlp(x, far, wts, e.gate_up_proj, e.down_proj)
        assert torch.equal(y, dense.experts_mlp(x, near, wts, e.gate_up_proj, e.down_proj)) and not y[1].any() and y[0].any()
